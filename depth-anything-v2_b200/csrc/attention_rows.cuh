// What the kernels of the grouped-head attention entries share: the parameters,
// the place of a row, the exact conversion of int8 codes to f16.
#pragma once

#include "kernels.cuh"

namespace dav2cuda {

constexpr uint32_t kMaxSplits = 128;

struct RowsParams {
    void* out;
    const void* q;
    const void* k;
    const void* v;
    const float* k_scales;
    const float* v_scales;
    const int32_t* page_table;
    const int32_t* lengths;      // keys of each sequence (null: all)
    const int32_t* query_begin;  // null: sequence s has rows [s * queries, (s + 1) * queries)
    uint64_t q_batch, q_stride, k_batch, k_stride, v_batch, v_stride, out_batch, out_stride;
    uint32_t sequences, queries, max_length, group, kv_heads, head_dim, pages, page_shift, table_stride;
    uint32_t causal, row_warps, splits, clusters, q_bf16, out_kind;  // out_kind: 0 f32, 1 bf16, 2 f16
    float scale_log2;
    // clusters: the splits of a row tile are the blocks of a cluster and join there
    float* part_o;   // [query][head][split][head_dim]
    float2* part_ml; // [query][head][split]
    int* err;
};

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) { return __byte_perm(a, b, s); }

__device__ __forceinline__ uint32_t hsub2_1152(uint32_t x) {
    uint32_t y;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
    return y;
}
// Codes in bytes 0, 1 (2, 3) of x, offset by 128, as two f16 values.
__device__ __forceinline__ uint32_t codes_lo(uint32_t x) { return hsub2_1152(prmt(x, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t codes_hi(uint32_t x) { return hsub2_1152(prmt(x, 0x64646464u, 0x4342)); }

// The V scale of a page as 2^e f, f in [1, 2). 2^e is added to the exponent of its keys, so that the
// running maximum, and what f16 holds of the weights, goes by p 2^e of the keys that the row itself
// sees: neither a page behind its mask nor one that it gives no weight takes bits from the others,
// however large its scale. f multiplies the weight, back = 2^-e brings it to p for the sum; all exact.
// Scales below 2^-90 leave the rest in f, which keeps 2^(7 - e) times 2^31 keys within f32.
__device__ __forceinline__ void split_scale(float scale, float& e, float& f, float& back) {
    const int i = max(-90, min(126, (int)(__float_as_uint(scale) >> 23) - 127));
    e = (float)i;
    back = __uint_as_float((uint32_t)(127 - i) << 23);
    f = scale * back;
}

template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (kBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

__device__ __forceinline__ float2 unpack2(uint32_t x, bool bf16) {
    if (bf16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

__device__ __forceinline__ void store_out(const RowsParams& p, uint64_t at, const float* x, uint32_t n) {
    if (p.out_kind == 0) {
        float* o = static_cast<float*>(p.out) + at;
        for (uint32_t i = 0; i < n; i += 2) *reinterpret_cast<float2*>(o + i) = make_float2(x[i], x[i + 1]);
    } else {
        uint16_t* o = static_cast<uint16_t*>(p.out) + at;
        for (uint32_t i = 0; i < n; i += 2)
            *reinterpret_cast<uint32_t*>(o + i) =
                p.out_kind == 1 ? pack2<true>(x[i], x[i + 1]) : pack2<false>(x[i], x[i + 1]);
    }
}

// The sequence, query rows and row tile of a block: sequence s has the blocks from
// floor(query_begin[s] * group / tile_rows) + s on, which leaves room for its rows
// whatever the lengths, so that the host needs none. False: no rows, or (error
// word 3) offsets out of range.
struct RowTile {
    uint32_t seq, q_begin, q_count, rows, tile;
};

__device__ __forceinline__ bool find_row_tile(RowTile& f, const RowsParams& p, uint32_t block, uint32_t tile_rows) {
    if (p.query_begin) {
        const uint32_t s = warp_last_at_most(p.sequences, block, [&](uint32_t i) {
            return (uint64_t)(uint32_t)p.query_begin[i] * p.group / tile_rows + i;
        });
        const int32_t b = p.query_begin[s], e = p.query_begin[s + 1];
        if (b < 0 || e < b || (uint32_t)e > p.queries) {
            if (threadIdx.x == 0) atomicExch(p.err, 3);
            return false;
        }
        const uint64_t first = (uint64_t)b * p.group / tile_rows + s;
        if (block < first) return false;
        f.seq = s, f.q_begin = b, f.q_count = e - b, f.tile = (uint32_t)(block - first);
    } else {
        const uint32_t tiles = (p.queries * p.group + tile_rows - 1) / tile_rows;
        f.seq = block / tiles;
        f.tile = block - f.seq * tiles;
        f.q_begin = 0, f.q_count = p.queries;
    }
    f.rows = f.q_count * p.group;
    return (uint64_t)f.tile * tile_rows < f.rows;
}

// Keys of a sequence, within max_length (else cut, error word 3).
__device__ __forceinline__ uint32_t keys_of(const RowsParams& p, uint32_t seq) {
    if (!p.lengths) return p.max_length;
    const int32_t length = p.lengths[seq];
    if (length < 0 || (uint32_t)length > p.max_length) {
        if (threadIdx.x == 0) atomicExch(p.err, 3);
        return length < 0 ? 0 : p.max_length;
    }
    return (uint32_t)length;
}

// Keys that a row sees; row = query * group + head within the key head's group.
__device__ __forceinline__ uint32_t reach_of(const RowsParams& p, const RowTile& f, uint32_t len, uint32_t row) {
    if (row >= f.rows) return 0;
    if (!p.causal) return len;
    const int64_t r = (int64_t)len - f.q_count + row / p.group + 1;
    return r > 0 ? (uint32_t)r : 0;
}

// Element of a live row in q or the output.
__device__ __forceinline__ uint64_t row_at(const RowsParams& p, const RowTile& f, uint32_t kv_head, uint32_t row,
                                           uint64_t batch, uint64_t stride) {
    const uint32_t i = row / p.group;
    const uint32_t head = kv_head * p.group + row - i * p.group;
    return (p.query_begin ? 0 : f.seq * batch) + ((uint64_t)f.q_begin + i) * stride + (uint64_t)head * p.head_dim;
}

// Slot of a live row's split in the workspace.
__device__ __forceinline__ uint64_t part_at(const RowsParams& p, const RowTile& f, uint32_t kv_head, uint32_t row,
                                            uint32_t split) {
    const uint32_t i = row / p.group;
    const uint64_t token = (p.query_begin ? 0ull : (uint64_t)f.seq * p.queries) + f.q_begin + i;
    return (token * (p.kv_heads * p.group) + kv_head * p.group + row - i * p.group) * p.splits + split;
}

// Rows kernel (attention_rows.cu): row tiles of 8 * row_tiles * p.row_warps rows.
int launch_attention_rows(const RowsParams& p, uint32_t slots, uint32_t row_tiles, bool s8, bool bf16,
                          cudaStream_t st);
// Tiles kernel (attention_tiles.cu): row tiles of 256 rows.
int launch_attention_tiles(const RowsParams& p, uint32_t slots, bool s8, bool bf16, cudaStream_t st);
// Joins the p.splits parts of each row.
int launch_attention_join(const RowsParams& p, uint64_t rows, cudaStream_t st);

}  // namespace dav2cuda

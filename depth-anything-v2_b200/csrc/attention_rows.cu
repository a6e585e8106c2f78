// Attention of a few query rows over many keys, for two sources of keys and
// values: the paged cache of int8 codes (one scale for each page and head) and
// 16-bit rows.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale * log2(e)
//
// in one pass with the running maximum m and sum of the softmax.
//
// The rows of one key head (query tokens x query heads that share it) are taken
// in tiles of 8 * NT as the N side of mma.m16n8k16, and keys, and then value
// dims, as its M side:
//   S^T[16 keys x 8 rows] = K[16 x d] Q^T[d x 8],  O^T[d x 8] += V^T[d x 16] P^T[16 x 8]
// so that one query token with up to eight query heads to a key head wastes
// nothing of the tile. Bound by memory for such rows: the tensor work is then a
// few percent, and what counts is bytes in flight. Keys and values go straight
// from global memory to the registers that the products need: the order of dims
// in q.k and of keys in p.v is free, so each lane loads 16 (8) consecutive bytes
// of a row and calls them its fragments. S^T's keys are laid so that transposing
// P's 8x8 blocks across lanes (movmatrix) gives the second product's operand.
//
// Codes become f16 exactly (byte + 1024 by a byte permutation, minus 1152), and q
// is scaled by a power of two for each row into f16's range, which keeps every
// bit of a bf16 or f16 value within 2^-29 of the row's largest. A K scale multiplies the
// scores of its 16 keys; a V scale multiplies p before it is rounded to f16,
// relative to the largest V scale R that the warp has met (O is kept in units of
// R and rescaled when R grows). p is at most 2^8 (m follows the row's maximum
// only when that exceeds it by 8) and is kept times 2^7, so that f16 holds
// contributions down to 2^-31 of the largest. The sum of p is kept in f32 from
// the unrounded values. 16-bit values take p in their own type, as the tensor
// core wants both operands alike.
//
// A block's four warps take either the same rows and every fourth 32 keys, merged
// at the end in shared memory, or (many rows) four row tiles and the same keys, which
// they then find in L1. Where there are few row tiles, the keys of a tile are split
// over several blocks whose (o, m, sum) go to the workspace, and a second kernel joins them.
#include <algorithm>
#include <cmath>

#include "abi_check.h"
#include "kernels.cuh"

namespace dav2cuda {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kChunk = 32;   // keys of one step of a warp
constexpr float kRaise = 8.0f;    // m is raised when a score exceeds it by this

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
    uint32_t causal, row_warps, splits, q_bf16, out_kind;  // out_kind: 0 f32, 1 bf16, 2 f16
    float scale_log2;
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

template <bool kBF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    if constexpr (kBF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
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

// One 16-key tile of codes or of 16-bit rows in registers.
template <int D, bool kS8>
struct Tile {
    static constexpr int kK = kS8 ? D / 64 : D / 32;                 // 16-byte loads of a K row
    static constexpr int kV = kS8 ? (D == 128 ? 4 : 2) : D / 16;     // words of a V row
    uint4 k[2][kK];
    uint32_t v[4][kV];
    float sk, sv;
    bool dead;  // no page of the cache: its keys are left out
};

struct Where {
    uint32_t seq, kv_head, len;   // len: keys of the sequence
};

template <int D, bool kS8>
__device__ __forceinline__ void load_tile(Tile<D, kS8>& f, const RowsParams& p, const Where& w, uint32_t key0,
                                          uint32_t lane) {
    const uint32_t g = lane >> 2, t = lane & 3, d = p.head_dim;
    const uint32_t kr = key0 + 4 * (g >> 1) + (g & 1);  // S^T row g is key kr, row g + 8 key kr + 2
    f.dead = false;
    if constexpr (kS8) {
        f.sk = f.sv = 0.0f;
        int32_t page = -1;
        if (key0 < w.len) {
            page = p.page_table[(uint64_t)w.seq * p.table_stride + (key0 >> p.page_shift)];
            if (page < 0 || (uint32_t)page >= p.pages) {
                if (lane == 0) atomicExch(p.err, 3);
                page = -1;
            }
        }
        if (page < 0) {
            f.dead = true;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < f.kK; ++i) f.k[h][i] = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < f.kV; ++j) f.v[i][j] = 0;
            return;
        }
        const uint64_t unit = (uint64_t)page * p.kv_heads + w.kv_head;
        f.sk = p.k_scales[unit], f.sv = p.v_scales[unit];
        const uint32_t in_page = (1u << p.page_shift) - 1;
        const uint64_t base = (unit << p.page_shift) * d;
        const int8_t* k = static_cast<const int8_t*>(p.k) + base;
        const int8_t* v = static_cast<const int8_t*>(p.v) + base;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < f.kK; ++i) {
                const uint32_t at = 64 * i + 16 * t;
                f.k[h][i] = at < d ? *reinterpret_cast<const uint4*>(k + ((kr + 2 * h) & in_page) * d + at)
                                   : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int8_t* row = v + ((key0 + 4 * t + i) & in_page) * d;
            if constexpr (D == 128) {
                const uint4 x = 16 * g < d ? *reinterpret_cast<const uint4*>(row + 16 * g) : make_uint4(0, 0, 0, 0);
                f.v[i][0] = x.x, f.v[i][1] = x.y, f.v[i][2] = x.z, f.v[i][3] = x.w;
            } else {
                const uint2 x = 8 * g < d ? *reinterpret_cast<const uint2*>(row + 8 * g) : make_uint2(0, 0);
                f.v[i][0] = x.x, f.v[i][1] = x.y;
            }
        }
    } else {
        f.sk = f.sv = 1.0f;
        const uint16_t* k = static_cast<const uint16_t*>(p.k) + w.seq * p.k_batch + (uint64_t)w.kv_head * d;
        const uint16_t* v = static_cast<const uint16_t*>(p.v) + w.seq * p.v_batch + (uint64_t)w.kv_head * d;
        // rows past the end are not read: they may be no memory, or hold NaN
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < f.kK; ++i) {
                const uint32_t at = 32 * i + 8 * t, key = kr + 2 * h;
                f.k[h][i] = at < d && key < w.len
                                ? *reinterpret_cast<const uint4*>(k + key * p.k_stride + at)
                                : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < f.kV; j += 4) {
                const uint32_t at = D / 8 * g + 2 * j, key = key0 + 4 * t + i;
                const uint4 x = at < d && key < w.len ? *reinterpret_cast<const uint4*>(v + key * p.v_stride + at)
                                                      : make_uint4(0, 0, 0, 0);
                f.v[i][j] = x.x, f.v[i][j + 1] = x.y, f.v[i][j + 2] = x.z, f.v[i][j + 3] = x.w;
            }
    }
}

__device__ __forceinline__ uint32_t word(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// kBF16: type of the second product's operands (false for codes).
template <int D, int NT, bool kS8, bool kBF16>
__global__ void __launch_bounds__(kThreads) attention_rows_kernel(const RowsParams p) {
    constexpr int kSteps = D / 16;
    constexpr int R = 8 * NT;
    __shared__ float s_o[kWarps][R][D + 4];
    __shared__ float s_m[kWarps][R], s_l[kWarps][R];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t tile_rows = R * p.row_warps, key_warps = kWarps / p.row_warps;
    const uint32_t row_warp = warp / key_warps, key_warp = warp % key_warps;

    // the sequence and the row tile of this block
    Where w;
    w.kv_head = blockIdx.y;
    uint32_t s = 0, q_begin, q_count, tile;
    if (p.query_begin) {
        for (uint32_t high = p.sequences; high - s > 1;) {
            const uint32_t mid = (s + high) / 2;
            if ((uint64_t)(uint32_t)p.query_begin[mid] * p.group / tile_rows + mid <= blockIdx.x) s = mid;
            else high = mid;
        }
        const int32_t b = p.query_begin[s], e = p.query_begin[s + 1];
        if (b < 0 || e < b || (uint32_t)e > p.queries) {
            if (threadIdx.x == 0) atomicExch(p.err, 3);
            return;
        }
        const uint64_t slot = (uint64_t)b * p.group / tile_rows + s;
        if (blockIdx.x < slot) return;
        q_begin = b, q_count = e - b;
        tile = (uint32_t)(blockIdx.x - slot);
    } else {
        const uint32_t tiles = (p.queries * p.group + tile_rows - 1) / tile_rows;
        s = blockIdx.x / tiles;
        tile = blockIdx.x - s * tiles;
        q_begin = 0, q_count = p.queries;
    }
    w.seq = s;
    const uint32_t rows = q_count * p.group;
    if ((uint64_t)tile * tile_rows >= rows) return;
    int32_t length = p.lengths ? p.lengths[s] : (int32_t)p.max_length;
    if (length < 0 || (uint32_t)length > p.max_length) {
        if (threadIdx.x == 0) atomicExch(p.err, 3);
        length = length < 0 ? 0 : (int32_t)p.max_length;
    }
    w.len = (uint32_t)length;
    const uint32_t row0 = tile * tile_rows + row_warp * R;  // this warp's first row

    auto reach_of = [&](uint32_t row) -> uint32_t {
        if (row >= rows) return 0;
        if (!p.causal) return w.len;
        const int64_t r = (int64_t)w.len - q_count + row / p.group + 1;
        return r > 0 ? (uint32_t)r : 0;
    };
    auto row_at = [&](uint32_t row, uint64_t batch, uint64_t stride) -> uint64_t {  // element of a live row
        const uint32_t i = row / p.group;
        const uint32_t head = w.kv_head * p.group + row - i * p.group;
        const uint64_t token = (uint64_t)q_begin + i;
        return (p.query_begin ? 0 : s * batch) + token * stride + (uint64_t)head * p.head_dim;
    };

    // q as the products' B fragments, and the factors of its rows
    uint32_t qf[NT][kSteps][2];
    float factor[NT][2];
    uint32_t reach[NT][2], low = 0xFFFFFFFFu, high = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const uint32_t row = row0 + 8 * n + g;
        const uint16_t* q = static_cast<const uint16_t*>(p.q) + (row < rows ? row_at(row, p.q_batch, p.q_stride) : 0);
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            // the dims of k-step j that the lane's K bytes hold
            const uint32_t at = kS8 ? 64 * (j / 4) + 16 * t + 4 * (j % 4) : 32 * (j / 2) + 8 * t + 4 * (j % 2);
            uint2 x = make_uint2(0, 0);
            if (row < rows && at < p.head_dim) x = *reinterpret_cast<const uint2*>(q + at);
            qf[n][j][0] = x.x, qf[n][j][1] = x.y;
            if constexpr (kS8) {
                const float2 a = unpack2(x.x, p.q_bf16), b = unpack2(x.y, p.q_bf16);
                most = fmaxf(fmaxf(most, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(b.x), fabsf(b.y)));
            }
        }
        float back = 1.0f;
        if constexpr (kS8) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            // 2^e brings the row's largest value into [2^14, 2^15); rows of zeros, and
            // exponents that would leave f32's range, stay near 1
            int e = most > 0.0f && most < INFINITY ? 141 - (int)(__float_as_uint(most) >> 23) : 0;
            e = max(-120, min(120, e));
            const float up = __uint_as_float((uint32_t)(127 + e) << 23);
            back = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
            for (int j = 0; j < kSteps; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 a = unpack2(qf[n][j][h], p.q_bf16);
                    qf[n][j][h] = pack2<false>(a.x * up, a.y * up);
                }
        }
        // lane g's row is column g of S^T; this lane's scores are columns 2t, 2t + 1
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            factor[n][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + e)) * p.scale_log2;
            reach[n][e] = reach_of(row0 + 8 * n + 2 * t + e);
            low = min(low, reach[n][e]);
            high = max(high, reach[n][e]);
        }
    }
#pragma unroll
    for (int o = 1; o < 4; o *= 2) {
        low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = max(high, __shfl_xor_sync(0xffffffffu, high, o));
    }

    // the keys of this split, in steps of kChunk, every key_warps-th for this warp
    const uint32_t chunks = (w.len + kChunk - 1) / kChunk;
    const uint32_t per_split = (chunks + p.splits - 1) / p.splits;
    const uint32_t first = blockIdx.z * per_split, last = min(chunks, first + per_split);

    float o[kSteps][NT][4], m[NT][2], l[NT][2], ref = 1e-30f, inv_ref = 128.0f / 1e-30f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
    }

    for (uint32_t c = first + key_warp; c < last; c += key_warps) {
        const uint32_t key0 = c * kChunk;
        if (key0 >= high) break;
        Tile<D, kS8> f[2];
        load_tile<D, kS8>(f[0], p, w, key0, lane);
        load_tile<D, kS8>(f[1], p, w, key0 + 16, lane);
        float sc[2][NT][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[b][n][0] = sc[b][n][1] = sc[b][n][2] = sc[b][n][3] = 0.0f;
            if constexpr (kS8) {
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    const uint32_t x = word(f[b].k[0][j / 4], j % 4) ^ 0x80808080u;
                    const uint32_t y = word(f[b].k[1][j / 4], j % 4) ^ 0x80808080u;
                    const uint32_t a0 = codes_lo(x), a1 = codes_lo(y), a2 = codes_hi(x), a3 = codes_hi(y);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816<false>(sc[b][n], a0, a1, a2, a3, qf[n][j][0], qf[n][j][1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    const uint4 &x = f[b].k[0][j / 2], &y = f[b].k[1][j / 2];
                    const int i = 2 * (j % 2);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        mma_16816<kBF16>(sc[b][n], word(x, i), word(y, i), word(x, i + 1), word(y, i + 1),
                                         qf[n][j][0], qf[n][j][1]);
                }
            }
        }
        // scores in units of log2, the keys out of reach at -inf
        bool raise = false;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[b][n][e] *= factor[n][e & 1] * f[b].sk;
        if (key0 + kChunk > low || f[0].dead || f[1].dead) {
            const uint32_t key = key0 + 4 * (g >> 1) + (g & 1);
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (f[b].dead || key + 16 * b + (e >= 2 ? 2 : 0) >= reach[n][e & 1]) sc[b][n][e] = -INFINITY;
        }
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[n][e] = fmaxf(fmaxf(sc[0][n][e], sc[0][n][e + 2]), fmaxf(sc[1][n][e], sc[1][n][e + 2]));
                raise |= top[n][e] > m[n][e] + kRaise;
            }
        const float sv_top = fmaxf(f[0].sv, f[1].sv);
        if (__any_sync(0xffffffffu, raise) || (kS8 && sv_top > ref)) {
            float unit = 1.0f;
            if (kS8 && sv_top > ref) {
                unit = ref / sv_top;
                ref = sv_top;
                inv_ref = 128.0f / ref;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = top[n][e];
#pragma unroll
                    for (int k = 4; k < 32; k *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, k));
                    x = fmaxf(x, m[n][e]);
                    const float down = x == -INFINITY ? 1.0f : ex2_approx(m[n][e] - x);
                    m[n][e] = x;
                    l[n][e] *= down;
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) o[i][n][e] *= down * unit, o[i][n][e + 2] *= down * unit;
                }
        }
        uint32_t pf[2][NT][2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const float weight = kS8 ? f[b].sv * inv_ref : kBF16 ? 1.0f : 128.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float e4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float mm = m[n][e & 1];
                    e4[e] = ex2_approx(sc[b][n][e] - (mm == -INFINITY ? 0.0f : mm));
                }
                l[n][0] += e4[0] + e4[2];
                l[n][1] += e4[1] + e4[3];
                pf[b][n][0] = transpose8x8(pack2<kBF16>(e4[0] * weight, e4[1] * weight));
                pf[b][n][1] = transpose8x8(pack2<kBF16>(e4[2] * weight, e4[3] * weight));
            }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const auto& v = f[b].v;
            if constexpr (kS8) {
#pragma unroll
                for (int i = 0; i < f[0].kV; ++i) {
                    const uint32_t x0 = v[0][i] ^ 0x80808080u, x1 = v[1][i] ^ 0x80808080u;
                    const uint32_t x2 = v[2][i] ^ 0x80808080u, x3 = v[3][i] ^ 0x80808080u;
                    const uint32_t l01 = prmt(x0, x1, 0x5140), h01 = prmt(x0, x1, 0x7362);
                    const uint32_t l23 = prmt(x2, x3, 0x5140), h23 = prmt(x2, x3, 0x7362);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_16816<false>(o[2 * i][n], codes_lo(l01), codes_hi(l01), codes_lo(l23), codes_hi(l23),
                                         pf[b][n][0], pf[b][n][1]);
                        mma_16816<false>(o[2 * i + 1][n], codes_lo(h01), codes_hi(h01), codes_lo(h23), codes_hi(h23),
                                         pf[b][n][0], pf[b][n][1]);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < f[0].kV; ++i) {
                    const uint32_t a0 = prmt(v[0][i], v[1][i], 0x5410), a1 = prmt(v[0][i], v[1][i], 0x7632);
                    const uint32_t a2 = prmt(v[2][i], v[3][i], 0x5410), a3 = prmt(v[2][i], v[3][i], 0x7632);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816<kBF16>(o[i][n], a0, a1, a2, a3, pf[b][n][0], pf[b][n][1]);
                }
            }
        }
    }

    // this warp's result: sums over the lanes that share a column, O in true units
    const float unit = kS8 ? ref * (1.0f / 128.0f) : kBF16 ? 1.0f : 1.0f / 128.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int k = 4; k < 32; k *= 2) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], k);
            const uint32_t col = 8 * n + 2 * t + e;
            if (g == 0) s_m[warp][col] = m[n][e], s_l[warp][col] = l[n][e];
            // tile i's rows g and g + 8 are dims D/8 g + 2i and the next
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
                *reinterpret_cast<float2*>(&s_o[warp][col][D / 8 * g + 2 * i]) =
                    make_float2(o[i][n][e] * unit, o[i][n][e + 2] * unit);
        }
    __syncthreads();

    // merge the key warps of each row tile: a thread takes two dims of a row
    for (uint32_t i = threadIdx.x; i < R * p.row_warps * (D / 2); i += kThreads) {
        const uint32_t r = i / (D / 2), dim = 2 * (i - r * (D / 2));
        const uint32_t rw = r / R, col = r - rw * R, row = tile * tile_rows + r;
        if (row >= rows || dim >= p.head_dim) continue;
        float top = -INFINITY;
        for (uint32_t k = 0; k < key_warps; ++k) top = fmaxf(top, s_m[rw * key_warps + k][col]);
        float sum = 0.0f, x[2] = {0.0f, 0.0f};
        for (uint32_t k = 0; k < key_warps; ++k) {
            const uint32_t kw = rw * key_warps + k;
            if (s_m[kw][col] == -INFINITY) continue;
            const float a = ex2_approx(s_m[kw][col] - top);
            sum += a * s_l[kw][col];
            x[0] += a * s_o[kw][col][dim];
            x[1] += a * s_o[kw][col][dim + 1];
        }
        if (p.splits == 1) {
            const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
            x[0] *= inv, x[1] *= inv;
            store_out(p, row_at(row, p.out_batch, p.out_stride) + dim, x, 2);
        } else {
            const uint32_t qi = row / p.group;
            const uint64_t token = (p.query_begin ? 0ull : (uint64_t)s * p.queries) + q_begin + qi;
            const uint64_t slot = (token * (p.kv_heads * p.group) + w.kv_head * p.group + row - qi * p.group) *
                                      p.splits + blockIdx.z;
            if (dim == 0) p.part_ml[slot] = make_float2(top, sum);
            if (sum > 0.0f) *reinterpret_cast<float2*>(p.part_o + slot * p.head_dim + dim) = make_float2(x[0], x[1]);
        }
    }
}

// Joins the splits of each row: a warp to a row.
__global__ void __launch_bounds__(kThreads) attention_join_kernel(const RowsParams p) {
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t row = (uint64_t)blockIdx.x * kWarps + threadIdx.x / 32;
    const uint32_t heads = p.kv_heads * p.group;
    const uint64_t token = row / heads;
    const uint64_t tokens = p.query_begin ? p.queries : (uint64_t)p.sequences * p.queries;
    if (token >= tokens) return;
    // rows of no sequence stay as they were
    if (p.query_begin && ((int64_t)token < p.query_begin[0] || (int64_t)token >= p.query_begin[p.sequences])) return;
    const uint32_t head = (uint32_t)(row - token * heads);
    const float2* ml = p.part_ml + row * p.splits;
    float top = -INFINITY;
    for (uint32_t k = lane; k < p.splits; k += 32) top = fmaxf(top, ml[k].x);
    top = warp_max(top);
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
    const uint32_t dim = 4 * lane;
    for (uint32_t k = 0; k < p.splits; ++k) {
        const float2 a = ml[k];
        if (!(a.y > 0.0f)) continue;
        const float f = ex2_approx(a.x - top);
        sum += f * a.y;
        if (dim < p.head_dim) {
            const float4 o = *reinterpret_cast<const float4*>(p.part_o + (row * p.splits + k) * p.head_dim + dim);
            x[0] += f * o.x, x[1] += f * o.y, x[2] += f * o.z, x[3] += f * o.w;
        }
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= inv;
    const uint64_t batch = p.query_begin ? 0 : token / p.queries;
    const uint64_t at = batch * p.out_batch + (token - batch * p.queries) * p.out_stride + (uint64_t)head * p.head_dim;
    const uint64_t flat = token * p.out_stride + (uint64_t)head * p.head_dim;
    if (dim < p.head_dim) store_out(p, (p.query_begin ? flat : at) + dim, x, 4);
}

struct Plan {
    uint32_t row_tiles;  // 8-row tiles of a warp
    uint32_t row_warps;
    uint32_t splits;
    uint64_t slots;
};

// Rows that share a key head decide the tile; the keys are split where the row
// tiles alone would leave SMs idle, down to 256 keys to a block.
Plan plan_rows(uint64_t sequences, uint64_t queries, bool ragged, uint32_t max_length, uint32_t group,
               uint32_t kv_heads, uint32_t sms) {
    Plan n;
    const uint64_t each = ragged ? (queries + sequences - 1) / sequences : queries;
    const uint64_t rows = each * group;
    n.row_tiles = rows <= 8 ? 1 : 2;
    n.row_warps = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    const uint64_t tile = 8ull * n.row_tiles * n.row_warps;
    n.slots = ragged ? queries * group / tile + sequences : sequences * ((rows + tile - 1) / tile);
    const uint64_t live = std::max<uint64_t>(1, sequences * ((rows + tile - 1) / tile)) * kv_heads;
    const uint64_t want = (3ull * sms + live - 1) / live;
    const uint64_t most = std::max<uint64_t>(1, max_length / 256);
    n.splits = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(want, most), 128);
    return n;
}

uint64_t workspace_of(const Plan& n, uint64_t tokens, uint32_t heads, uint32_t head_dim) {
    if (n.splits == 1) return 0;
    return tokens * heads * n.splits * (head_dim * 4ull + 8) + 256;
}

template <int D, int NT, bool kS8, bool kBF16>
void start(const RowsParams& p, const Plan& n, cudaStream_t st) {
    attention_rows_kernel<D, NT, kS8, kBF16>
        <<<dim3((uint32_t)n.slots, p.kv_heads, n.splits), kThreads, 0, st>>>(p);
}

template <bool kS8, bool kBF16>
void start_for(const RowsParams& p, const Plan& n, cudaStream_t st) {
    if (p.head_dim <= 64) {
        if (n.row_tiles == 1) start<64, 1, kS8, kBF16>(p, n, st);
        else start<64, 2, kS8, kBF16>(p, n, st);
    } else {
        if (n.row_tiles == 1) start<128, 1, kS8, kBF16>(p, n, st);
        else start<128, 2, kS8, kBF16>(p, n, st);
    }
}

int run_rows(RowsParams& p, const Plan& n, bool s8, bool bf16, uint64_t tokens, void* workspace, cudaStream_t st) {
    p.row_warps = n.row_warps, p.splits = n.splits;
    if (n.splits > 1) {
        const uint64_t slots = tokens * p.kv_heads * p.group * n.splits;
        uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~uintptr_t(15));
        p.part_o = reinterpret_cast<float*>(base);
        p.part_ml = reinterpret_cast<float2*>(base + slots * p.head_dim * 4);
    }
    if (s8) start_for<true, false>(p, n, st);
    else if (bf16) start_for<false, true>(p, n, st);
    else start_for<false, false>(p, n, st);
    if (int rc = check_launch("attention_rows")) return rc;
    if (n.splits == 1) return DAV2CUDA_OK;
    const uint64_t rows = tokens * p.kv_heads * p.group;
    attention_join_kernel<<<(uint32_t)((rows + kWarps - 1) / kWarps), kThreads, 0, st>>>(p);
    return check_launch("attention_join");
}

bool shape_ok(uint32_t q_heads, uint32_t kv_heads) {
    return q_heads >= 1 && kv_heads >= 1 && kv_heads <= 65535 && q_heads % kv_heads == 0 && q_heads <= 65535;
}

}  // namespace
}  // namespace dav2cuda

using namespace dav2cuda;

// The sizes are answered for 148 SMs, a B200's, so that they need no device.
constexpr uint32_t kPlanSms = 148;

extern "C" DAV2CUDA_API uint64_t dav2cuda_attention_cache_s8_workspace_size(uint32_t sequences, uint32_t queries,
                                                                            uint32_t max_length, uint32_t q_heads,
                                                                            uint32_t kv_heads, uint32_t head_dim) {
    if (!sequences || !queries || !shape_ok(q_heads, kv_heads)) return 0;
    const Plan n = plan_rows(sequences, queries, true, max_length, q_heads / kv_heads, kv_heads, kPlanSms);
    return workspace_of(n, queries, q_heads, head_dim);
}

extern "C" DAV2CUDA_API int dav2cuda_attention_cache_s8(
    void* output, const void* q, const int8_t* k_codes, const float* k_scales, const int8_t* v_codes,
    const float* v_scales, const int32_t* page_table, const int32_t* lengths, const int32_t* query_begin,
    uint32_t sequences, uint32_t queries, uint32_t max_length, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,
    uint32_t page_count, uint32_t page_tokens, uint32_t table_stride, uint64_t q_stride, uint64_t output_stride,
    float scale, uint32_t causal, uint32_t precision, uint32_t output_precision, void* workspace,
    uint64_t workspace_bytes, void* stream) {
    DAV2_REQUIRE(precision == 1 || precision == 2, "cache attention: queries must be bf16 or f16");
    DAV2_REQUIRE(output_precision == 0 || output_precision == precision,
                 "cache attention: output must be f32 or of the queries' type");
    DAV2_REQUIRE(shape_ok(q_heads, kv_heads), "cache attention: q_heads must be a multiple of kv_heads");
    DAV2_REQUIRE(head_dim >= 16 && head_dim <= 128 && head_dim % 16 == 0,
                 "cache attention: head_dim must be a multiple of 16, 16 to 128");
    DAV2_REQUIRE(page_tokens >= 16 && page_tokens <= 128 && (page_tokens & (page_tokens - 1)) == 0,
                 "cache attention: page_tokens must be 16, 32, 64 or 128");
    DAV2_REQUIRE(page_count >= 1 && page_count <= 0x7FFFFFFFu && table_stride >= 1 && max_length <= 0x7FFFFF00u &&
                     (uint64_t)table_stride * page_tokens >= max_length,
                 "cache attention: the page table does not hold max_length tokens");
    DAV2_REQUIRE(std::isfinite(scale), "cache attention: invalid scale");
    DAV2_REQUIRE((uint64_t)queries * (q_heads / kv_heads) <= 0x3FFFFFFFu && sequences <= 0x3FFFFFFFu,
                 "cache attention: too many queries or sequences");
    if (!queries || !sequences) return DAV2CUDA_OK;
    const uint64_t row = (uint64_t)q_heads * head_dim;
    DAV2_REQUIRE(queries == 1 || (q_stride >= row && output_stride >= row),
                 "cache attention: a token stride is below the row of its heads");
    DAV2_REQUIRE(!any_null(output, q, k_codes, k_scales, v_codes, v_scales, page_table, lengths, query_begin),
                 "cache attention: null buffer");
    DAV2_REQUIRE(aligned16(output) && aligned16(q) && aligned16(k_codes) && aligned16(v_codes) &&
                     (queries == 1 || (q_stride % 8 == 0 && output_stride % 8 == 0)),
                 "cache attention: rows must be 16-byte aligned");
    RowsParams p{};
    p.out = output, p.q = q, p.k = k_codes, p.v = v_codes, p.k_scales = k_scales, p.v_scales = v_scales;
    p.page_table = page_table, p.lengths = lengths, p.query_begin = query_begin;
    p.q_stride = q_stride, p.out_stride = output_stride;
    p.sequences = sequences, p.queries = queries, p.max_length = max_length, p.group = q_heads / kv_heads;
    p.kv_heads = kv_heads, p.head_dim = head_dim, p.pages = page_count, p.table_stride = table_stride;
    p.page_shift = 4;
    while ((1u << p.page_shift) < page_tokens) ++p.page_shift;
    p.causal = causal != 0, p.q_bf16 = precision == 1, p.out_kind = output_precision;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634);
    const Plan n = plan_rows(sequences, queries, true, max_length, p.group, kv_heads, kPlanSms);
    DAV2_REQUIRE(n.slots <= 0x7FFFFFFFu, "cache attention: too many queries or sequences");
    const uint64_t need = workspace_of(n, queries, q_heads, head_dim);
    DAV2_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "cache attention: workspace is too small");
    p.err = device_error_word();
    if (!p.err) return set_error(DAV2CUDA_INTERNAL_ERROR, "cache attention: no device error word");
    return run_rows(p, n, true, false, queries, workspace, as_stream(stream));
}

extern "C" DAV2CUDA_API uint64_t dav2cuda_cross_attention_16_workspace_size(uint32_t batch, uint32_t queries,
                                                                            uint32_t keys, uint32_t q_heads,
                                                                            uint32_t kv_heads, uint32_t head_dim) {
    if (!batch || !queries || !shape_ok(q_heads, kv_heads)) return 0;
    const Plan n = plan_rows(batch, queries, false, keys, q_heads / kv_heads, kv_heads, kPlanSms);
    return workspace_of(n, (uint64_t)batch * queries, q_heads, head_dim);
}

extern "C" DAV2CUDA_API int dav2cuda_cross_attention_16(
    void* output, const void* q, const void* k, const void* v, const int32_t* key_lengths, uint32_t batch,
    uint32_t queries, uint32_t keys, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint64_t q_batch_stride,
    uint64_t q_stride, uint64_t k_batch_stride, uint64_t k_stride, uint64_t v_batch_stride, uint64_t v_stride,
    uint64_t output_batch_stride, uint64_t output_stride, float scale, uint32_t precision, uint32_t output_precision,
    void* workspace, uint64_t workspace_bytes, void* stream) {
    DAV2_REQUIRE(precision == 1 || precision == 2, "cross attention: operands must be bf16 or f16");
    DAV2_REQUIRE(output_precision == 0 || output_precision == precision,
                 "cross attention: output must be f32 or of the operands' type");
    DAV2_REQUIRE(shape_ok(q_heads, kv_heads), "cross attention: q_heads must be a multiple of kv_heads");
    DAV2_REQUIRE(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0,
                 "cross attention: head_dim must be a multiple of 8, 8 to 128");
    DAV2_REQUIRE(std::isfinite(scale), "cross attention: invalid scale");
    DAV2_REQUIRE((uint64_t)batch * queries * (q_heads / kv_heads) <= 0x3FFFFFFFu && keys <= 0x7FFFFF00u,
                 "cross attention: too many queries or keys");
    if (!queries || !batch) return DAV2CUDA_OK;
    const uint64_t row = (uint64_t)q_heads * head_dim, kv_row = (uint64_t)kv_heads * head_dim;
    DAV2_REQUIRE(queries == 1 || (q_stride >= row && output_stride >= row),
                 "cross attention: a token stride is below the row of its heads");
    DAV2_REQUIRE(keys <= 1 || (k_stride >= kv_row && v_stride >= kv_row),
                 "cross attention: a token stride is below the row of its heads");
    DAV2_REQUIRE(batch == 1 || output_batch_stride >= (queries - 1) * output_stride + row,
                 "cross attention: output batches overlap");
    DAV2_REQUIRE(!any_null(output, q) && (keys == 0 || !any_null(k, v)), "cross attention: null buffer");
    DAV2_REQUIRE(aligned16(output) && aligned16(q) && aligned16(k) && aligned16(v) &&
                     (queries == 1 || (q_stride % 8 == 0 && output_stride % 8 == 0)) &&
                     (keys <= 1 || (k_stride % 8 == 0 && v_stride % 8 == 0)) &&
                     (batch == 1 || (q_batch_stride % 8 == 0 && output_batch_stride % 8 == 0 &&
                                     k_batch_stride % 8 == 0 && v_batch_stride % 8 == 0)),
                 "cross attention: rows must be 16-byte aligned");
    RowsParams p{};
    p.out = output, p.q = q, p.k = k, p.v = v, p.lengths = key_lengths;
    p.q_batch = q_batch_stride, p.q_stride = q_stride, p.k_batch = k_batch_stride, p.k_stride = k_stride;
    p.v_batch = v_batch_stride, p.v_stride = v_stride, p.out_batch = output_batch_stride, p.out_stride = output_stride;
    p.sequences = batch, p.queries = queries, p.max_length = keys, p.group = q_heads / kv_heads;
    p.kv_heads = kv_heads, p.head_dim = head_dim, p.q_bf16 = precision == 1, p.out_kind = output_precision;
    p.scale_log2 = (float)((double)scale * 1.4426950408889634);
    const Plan n = plan_rows(batch, queries, false, keys, p.group, kv_heads, kPlanSms);
    DAV2_REQUIRE(n.slots <= 0x7FFFFFFFu, "cross attention: too many queries");
    const uint64_t tokens = (uint64_t)batch * queries, need = workspace_of(n, tokens, q_heads, head_dim);
    DAV2_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "cross attention: workspace is too small");
    p.err = device_error_word();
    if (!p.err) return set_error(DAV2CUDA_INTERNAL_ERROR, "cross attention: no device error word");
    return run_rows(p, n, false, precision == 1, tokens, workspace, as_stream(stream));
}

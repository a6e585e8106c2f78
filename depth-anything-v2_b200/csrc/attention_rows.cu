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
// A block's four warps take either the same rows and every fourth step of keys, merged
// at the end in shared memory, or (many rows) four row tiles and the same keys, which
// they then find in L1. Where there are few row tiles, the keys of a tile are split
// over several blocks whose (o, m, sum) go to the workspace, and a second kernel joins them.
#include "attention_rows.cuh"

namespace dav2cuda {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr float kRaise = 8.0f;    // m is raised when a score exceeds it by this

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

__device__ __forceinline__ uint32_t word(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Address of a shared-memory place of this block in another block of the cluster.
__device__ __forceinline__ uint32_t cluster_place(const void* p, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
    return a;
}

__device__ __forceinline__ float cluster_load(uint32_t place) {
    float x;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(place) : "memory");
    return x;
}

__device__ __forceinline__ float2 cluster_load2(uint32_t place) {
    float2 x;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(place) : "memory");
    return x;
}

// The keys of one step of a warp in registers, as tiles of 16 (4 KB of codes or of
// 16-bit values at D = 128, K and V). S^T's row g of a tile is key 4 (g / 2) + g % 2, row g + 8 the second next; a lane's V rows are keys 4t .. 4t + 3.
// kFull: head_dim == D, known to the compiler.
template <int D, bool kS8, bool kFull>
struct Source {
    static constexpr int kTiles = kS8 ? 2 : 1;
    static constexpr uint32_t kChunk = 16 * kTiles;
    static constexpr int kK = kS8 ? D / 64 : D / 32;              // 16-byte loads of a K row
    static constexpr int kV = kS8 ? (D == 128 ? 4 : 2) : D / 16;  // words of a V row
    const RowsParams& p;
    uint32_t seq, kv_head, len, g, t, d;
    uint64_t at_k, at_v;                // this lane's place in a tile, 16-bit rows: in the batch entry
    uint4 k[kTiles][2][kK];                  // [tile][row][load]
    uint32_t v[kTiles][4][kV];          // [tile][key][word]
    float sk[kTiles], sv[kTiles];
    int32_t page_k[kTiles], page_v[kTiles], page_next[kTiles];  // of the tiles in k, in v, and of the chunk to come; -1: none

    __device__ Source(const RowsParams& p, uint32_t seq, uint32_t kv_head, uint32_t len, uint32_t lane)
        : p(p), seq(seq), kv_head(kv_head), len(len), g(lane >> 2), t(lane & 3), d(kFull ? D : p.head_dim) {
        const uint32_t kr = 4 * (g >> 1) + (g & 1);
        if constexpr (kS8) {
            at_k = kr * d + 16 * t;
            at_v = 4 * t * d + D / 8 * g;
        } else {
            at_k = seq * p.k_batch + (uint64_t)kv_head * d + kr * p.k_stride + 8 * t;
            at_v = seq * p.v_batch + (uint64_t)kv_head * d + 4 * t * p.v_stride + D / 8 * g;
        }
    }

    // The pages of the chunk at key0 (codes), fetched ahead of their use.
    __device__ __forceinline__ void fetch_pages(uint32_t key0) {
        if constexpr (kS8) {
#pragma unroll
            for (int b = 0; b < kTiles; ++b) {
                const uint32_t key = key0 + 16 * b;
                page_next[b] =
                    key < len ? p.page_table[(uint64_t)seq * p.table_stride + (key >> p.page_shift)] : -1;
            }
        }
    }

    __device__ __forceinline__ uint64_t tile_of(int32_t page, uint32_t key) const {
        const uint64_t unit = (uint64_t)(uint32_t)page * p.kv_heads + kv_head;
        return ((unit << p.page_shift) + (key & ((1u << p.page_shift) - 1))) * d;
    }

    __device__ __forceinline__ void load_k(uint32_t key0) {
        if constexpr (kS8) {
#pragma unroll
            for (int b = 0; b < kTiles; ++b) {
                const uint32_t key = key0 + 16 * b;
                int32_t page = page_next[b];
                if (page < 0 || (uint32_t)page >= p.pages) {
                    if (key < len && threadIdx.x % 32 == 0) atomicExch(p.err, 3);
                    page = -1;
                }
                page_k[b] = page;
                sk[b] = sv[b] = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < kK; ++i) k[b][h][i] = make_uint4(0, 0, 0, 0);
                if (page < 0) continue;
                const uint64_t unit = (uint64_t)(uint32_t)page * p.kv_heads + kv_head;
                sk[b] = p.k_scales[unit], sv[b] = p.v_scales[unit];
                const int8_t* from = static_cast<const int8_t*>(p.k) + tile_of(page, key) + at_k;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < kK; ++i)
                        if (kFull || 64 * i + 16 * t < d)
                            k[b][h][i] = *reinterpret_cast<const uint4*>(from + 2 * h * d + 64 * i);
            }
        } else {
            // rows past the end are not read: they may be no memory, or hold NaN
            const uint16_t* from = static_cast<const uint16_t*>(p.k) + at_k + key0 * p.k_stride;
            const uint32_t key = key0 + 4 * (g >> 1) + (g & 1);
#pragma unroll
            for (int b = 0; b < kTiles; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < kK; ++i)
                        k[b][h][i] = (kFull || 32 * i + 8 * t < d) && key + 16 * b + 2 * h < len
                                         ? *reinterpret_cast<const uint4*>(from + (16 * b + 2 * h) * p.k_stride + 32 * i)
                                         : make_uint4(0, 0, 0, 0);
        }
    }

    __device__ __forceinline__ void load_v(uint32_t key0) {
        if constexpr (kS8) {
#pragma unroll
            for (int b = 0; b < kTiles; ++b) {
                page_v[b] = page_k[b];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < kV; ++j) v[b][i][j] = 0;
                if (page_v[b] < 0 || !(kFull || D / 8 * g < d)) continue;
                const int8_t* from = static_cast<const int8_t*>(p.v) + tile_of(page_v[b], key0 + 16 * b) + at_v;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (D == 128) {
                        const uint4 x = *reinterpret_cast<const uint4*>(from + i * d);
                        v[b][i][0] = x.x, v[b][i][1] = x.y, v[b][i][2] = x.z, v[b][i][3] = x.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2*>(from + i * d);
                        v[b][i][0] = x.x, v[b][i][1] = x.y;
                    }
                }
            }
        } else {
            const uint16_t* from = static_cast<const uint16_t*>(p.v) + at_v + key0 * p.v_stride;
#pragma unroll
            for (int b = 0; b < kTiles; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < kV; j += 4) {
                        const uint4 x = (kFull || D / 8 * g + 2 * j < d) && key0 + 16 * b + 4 * t + i < len
                                            ? *reinterpret_cast<const uint4*>(from + (16 * b + i) * p.v_stride + 2 * j)
                                            : make_uint4(0, 0, 0, 0);
                        v[b][i][j] = x.x, v[b][i][j + 1] = x.y, v[b][i][j + 2] = x.z, v[b][i][j + 3] = x.w;
                    }
        }
    }
};

// kBF16: type of the second product's operands (false for codes).
template <int D, int NT, bool kS8, bool kBF16, bool kFull>
__global__ void __launch_bounds__(kThreads) attention_rows_kernel(const RowsParams p) {
    using Keys = Source<D, kS8, kFull>;
    constexpr int kSteps = D / 16, kTiles = Keys::kTiles;
    constexpr uint32_t kChunk = Keys::kChunk;
    constexpr int R = 8 * NT;
    __shared__ float s_o[kWarps][R][D + 4];
    __shared__ float s_m[kWarps][R], s_l[kWarps][R];
    __shared__ float c_m[kWarps * R], c_l[kWarps * R];  // of the block's rows, for the cluster
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t tile_rows = R * p.row_warps, key_warps = kWarps / p.row_warps;
    const uint32_t row_warp = warp / key_warps, key_warp = warp % key_warps;
    const uint32_t d = kFull ? D : p.head_dim;

    RowTile where;
    if (!find_row_tile(where, p, blockIdx.x, tile_rows)) return;
    const uint32_t kv_head = blockIdx.y, len = keys_of(p, where.seq), rows = where.rows;
    const uint32_t row0 = where.tile * tile_rows + row_warp * R;  // this warp's first row

    // the keys of this split, in steps of kChunk, every key_warps-th for this warp
    const uint32_t chunks = (len + kChunk - 1) / kChunk;
    const uint32_t per_split = (chunks + p.splits - 1) / p.splits;
    const uint32_t first = blockIdx.z * per_split;
    Keys f(p, where.seq, kv_head, len, lane);
    uint32_t c = first + key_warp;
    f.fetch_pages(c * kChunk);

    // q as the products' B fragments, and the factors of its rows
    uint32_t qf[NT][kSteps][2];
    float factor[NT][2];
    uint32_t reach[NT][2], low = 0xFFFFFFFFu, high = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const uint32_t row = row0 + 8 * n + g;
        const uint16_t* q = static_cast<const uint16_t*>(p.q) +
                            (row < rows ? row_at(p, where, kv_head, row, p.q_batch, p.q_stride) : 0);
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            // the dims of k-step j that the lane's K bytes hold
            const uint32_t at = kS8 ? 64 * (j / 4) + 16 * t + 4 * (j % 4) : 32 * (j / 2) + 8 * t + 4 * (j % 2);
            uint2 x = make_uint2(0, 0);
            if (row < rows && at < d) x = *reinterpret_cast<const uint2*>(q + at);
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
            reach[n][e] = reach_of(p, where, len, row0 + 8 * n + 2 * t + e);
            low = min(low, reach[n][e]);
            high = max(high, reach[n][e]);
        }
    }
#pragma unroll
    for (int o = 1; o < 4; o *= 2) {
        low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = max(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    const uint32_t last = min(min(chunks, first + per_split), (high + kChunk - 1) / kChunk);

    float o[kSteps][NT][4], m[NT][2], l[NT][2], ref = 1e-30f, inv_ref = 128.0f / 1e-30f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
    }

    // Two loads are in flight at any time: K of the next chunk from the first product
    // on, V of the next chunk from the second on, into the registers just used.
    if (c < last) {
        f.load_k(c * kChunk);
        f.load_v(c * kChunk);
        f.fetch_pages((c + key_warps) * kChunk);
    }
    for (; c < last; c += key_warps) {
        const uint32_t key0 = c * kChunk, next = (c + key_warps) * kChunk;
        const bool more = c + key_warps < last;
        float sc[kTiles][NT][4];
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[b][n][0] = sc[b][n][1] = sc[b][n][2] = sc[b][n][3] = 0.0f;
            if constexpr (kS8) {
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    const uint32_t x = word(f.k[b][0][j / 4], j % 4) ^ 0x80808080u;
                    const uint32_t y = word(f.k[b][1][j / 4], j % 4) ^ 0x80808080u;
                    const uint32_t a0 = codes_lo(x), a1 = codes_lo(y), a2 = codes_hi(x), a3 = codes_hi(y);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816<false>(sc[b][n], a0, a1, a2, a3, qf[n][j][0], qf[n][j][1]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    const uint4 &x = f.k[b][0][j / 2], &y = f.k[b][1][j / 2];
                    const int i = 2 * (j % 2);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        mma_16816<kBF16>(sc[b][n], word(x, i), word(y, i), word(x, i + 1), word(y, i + 1),
                                         qf[n][j][0], qf[n][j][1]);
                }
            }
        }
        float sk[kTiles], sv[kTiles], sv_top = 0.0f;
        bool dead[kTiles], any_dead = false;
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
            sk[b] = kS8 ? f.sk[b] : 1.0f, sv[b] = kS8 ? f.sv[b] : 1.0f;
            sv_top = fmaxf(sv_top, sv[b]);
            dead[b] = kS8 && f.page_k[b] < 0;
            any_dead |= dead[b];
        }
        if (more) f.load_k(next);
        // scores in units of log2, the keys out of reach at -inf
        bool raise = false;
#pragma unroll
        for (int b = 0; b < kTiles; ++b)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[b][n][e] *= kS8 ? factor[n][e & 1] * sk[b] : factor[n][e & 1];
        if (key0 + kChunk > low || any_dead) {
            const uint32_t key = key0 + 4 * (g >> 1) + (g & 1);
#pragma unroll
            for (int b = 0; b < kTiles; ++b)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (dead[b] || key + 16 * b + (e >= 2 ? 2 : 0) >= reach[n][e & 1]) sc[b][n][e] = -INFINITY;
        }
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[n][e] = fmaxf(sc[0][n][e], sc[0][n][e + 2]);
                if (kTiles == 2) top[n][e] = fmaxf(top[n][e], fmaxf(sc[kTiles - 1][n][e], sc[kTiles - 1][n][e + 2]));
                raise |= top[n][e] > m[n][e] + kRaise;
            }
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
        uint32_t pf[kTiles][NT][2];
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
            const float weight = kS8 ? sv[b] * inv_ref : kBF16 ? 1.0f : 128.0f;
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
        for (int b = 0; b < kTiles; ++b) {
            const auto& v = f.v[b];
            if constexpr (kS8) {
#pragma unroll
                for (int i = 0; i < f.kV; ++i) {
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
                for (int i = 0; i < f.kV; ++i) {
                    const uint32_t a0 = prmt(v[0][i], v[1][i], 0x5410), a1 = prmt(v[0][i], v[1][i], 0x7632);
                    const uint32_t a2 = prmt(v[2][i], v[3][i], 0x5410), a3 = prmt(v[2][i], v[3][i], 0x7632);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816<kBF16>(o[i][n], a0, a1, a2, a3, pf[b][n][0], pf[b][n][1]);
                }
            }
        }
        if (more) {
            f.load_v(next);
            f.fetch_pages(next + key_warps * kChunk);
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
    for (uint32_t i = threadIdx.x; i < tile_rows * (D / 2); i += kThreads) {
        const uint32_t r = i / (D / 2), dim = 2 * (i - r * (D / 2));
        const uint32_t w0 = r / R * key_warps, col = r % R, row = where.tile * tile_rows + r;
        if (row >= rows || dim >= d) continue;
        float top = -INFINITY;
        for (uint32_t k = 0; k < key_warps; ++k) top = fmaxf(top, s_m[w0 + k][col]);
        float sum = 0.0f, x[2] = {0.0f, 0.0f};
        for (uint32_t k = 0; k < key_warps; ++k) {
            if (s_m[w0 + k][col] == -INFINITY) continue;
            const float a = ex2_approx(s_m[w0 + k][col] - top);
            sum += a * s_l[w0 + k][col];
            const float2 b = *reinterpret_cast<const float2*>(&s_o[w0 + k][col][dim]);
            x[0] += a * b.x;
            x[1] += a * b.y;
        }
        if (p.splits == 1) {
            const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
            x[0] *= inv, x[1] *= inv;
            store_out(p, row_at(p, where, kv_head, row, p.out_batch, p.out_stride) + dim, x, 2);
        } else if (p.clusters) {
            *reinterpret_cast<float2*>(&s_o[w0][col][dim]) = make_float2(x[0], x[1]);  // read by this thread alone
            if (dim == 0) c_m[r] = top, c_l[r] = sum;
        } else {
            const uint64_t slot = part_at(p, where, kv_head, row, blockIdx.z);
            if (dim == 0) p.part_ml[slot] = make_float2(top, sum);
            if (sum > 0.0f) *reinterpret_cast<float2*>(p.part_o + slot * d + dim) = make_float2(x[0], x[1]);
        }
    }
    if (!p.clusters) return;
    // the splits are a cluster: each block merges its share of the rows' dims
    cluster_sync();
    for (uint32_t i = blockIdx.z * kThreads + threadIdx.x; i < tile_rows * (D / 2); i += p.splits * kThreads) {
        const uint32_t r = i / (D / 2), dim = 2 * (i - r * (D / 2));
        const uint32_t w0 = r / R * key_warps, col = r % R, row = where.tile * tile_rows + r;
        if (row >= rows || dim >= d) continue;
        float top = -INFINITY;
        for (uint32_t k = 0; k < p.splits; ++k) top = fmaxf(top, cluster_load(cluster_place(&c_m[r], k)));
        float sum = 0.0f, x[2] = {0.0f, 0.0f};
        for (uint32_t k = 0; k < p.splits; ++k) {
            const float mk = cluster_load(cluster_place(&c_m[r], k));
            if (mk == -INFINITY) continue;
            const float a = ex2_approx(mk - top);
            sum += a * cluster_load(cluster_place(&c_l[r], k));
            const float2 b = cluster_load2(cluster_place(&s_o[w0][col][dim], k));
            x[0] += a * b.x;
            x[1] += a * b.y;
        }
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        x[0] *= inv, x[1] *= inv;
        store_out(p, row_at(p, where, kv_head, row, p.out_batch, p.out_stride) + dim, x, 2);
    }
    cluster_sync();  // no block leaves while another reads its shared memory
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

template <int D, int NT, bool kS8, bool kBF16, bool kFull>
int start(const RowsParams& p, uint32_t slots, cudaStream_t st) {
    cudaLaunchAttribute cluster[1];
    cluster[0].id = cudaLaunchAttributeClusterDimension;
    cluster[0].val.clusterDim.x = 1, cluster[0].val.clusterDim.y = 1, cluster[0].val.clusterDim.z = p.splits;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(slots, p.kv_heads, p.splits);
    config.blockDim = dim3(kThreads);
    config.stream = st;
    config.attrs = cluster;
    config.numAttrs = p.clusters ? 1 : 0;
    cudaLaunchKernelEx(&config, attention_rows_kernel<D, NT, kS8, kBF16, kFull>, p);
    return check_launch("attention_rows");
}

template <bool kS8, bool kBF16>
int start_for(const RowsParams& p, uint32_t slots, uint32_t row_tiles, cudaStream_t st) {
    if (p.head_dim == 64) return row_tiles == 1 ? start<64, 1, kS8, kBF16, true>(p, slots, st)
                                                : start<64, 2, kS8, kBF16, true>(p, slots, st);
    if (p.head_dim == 128) return row_tiles == 1 ? start<128, 1, kS8, kBF16, true>(p, slots, st)
                                                 : start<128, 2, kS8, kBF16, true>(p, slots, st);
    if (p.head_dim < 64) return row_tiles == 1 ? start<64, 1, kS8, kBF16, false>(p, slots, st)
                                               : start<64, 2, kS8, kBF16, false>(p, slots, st);
    return row_tiles == 1 ? start<128, 1, kS8, kBF16, false>(p, slots, st)
                          : start<128, 2, kS8, kBF16, false>(p, slots, st);
}

}  // namespace

int launch_attention_rows(const RowsParams& p, uint32_t slots, uint32_t row_tiles, bool s8, bool bf16,
                          cudaStream_t st) {
    if (s8) return start_for<true, false>(p, slots, row_tiles, st);
    return bf16 ? start_for<false, true>(p, slots, row_tiles, st) : start_for<false, false>(p, slots, row_tiles, st);
}

int launch_attention_join(const RowsParams& p, uint64_t rows, cudaStream_t st) {
    attention_join_kernel<<<(uint32_t)((rows + kWarps - 1) / kWarps), kThreads, 0, st>>>(p);
    return check_launch("attention_join");
}

}  // namespace dav2cuda

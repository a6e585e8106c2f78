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
// few percent, and what counts is bytes in flight: each warp has a ring of keys and
// values in shared memory that it fills with asynchronous copies of its own, two (16-bit
// rows: three) steps of 16 or 32 keys deep, and waits for no other warp. The order of
// dims in q.k and of keys in p.v is free, so each lane reads 16 (8) consecutive bytes of
// a row from it and calls them its fragments. S^T's keys are laid so that transposing
// P's 8x8 blocks across lanes (movmatrix) gives the second product's operand.
//
// Codes become f16 exactly (byte + 1024 by a byte permutation, minus 1152), and q
// is scaled by a power of two for each row into f16's range, which keeps every
// bit of a bf16 or f16 value within 2^-29 of the row's largest. A K scale multiplies the
// scores of its 16 keys; a V scale 2^e f adds e to them and multiplies p by f before it
// is rounded to f16, so that m is the maximum of score + e: of what keys contribute, not
// of their scores alone. p is at most 2^7 (m follows the row's maximum only when that
// exceeds it by 7) and is kept times 2^7, so that f16 holds contributions down to 2^-31
// of the row's largest, whatever the scales of pages that it does not see or gives no
// weight. The sum takes p times 2^-e in f32, unrounded. 16-bit values take p in their own
// type, as the tensor core wants both operands alike (p at most 2^8).
//
// A block's four warps take the same rows and every fourth step of keys, or (more than 16
// rows) two row tiles and every second step, merged at the end in shared memory. Where
// there are few row tiles, the keys of a tile are split over several blocks: up to eight
// are a cluster that joins their (o, m, sum) over its shared memory; more go to the
// workspace, and a second kernel, launched before the first has ended, joins them.
//
// Codes: the conversion shares the issue slots with the loads (of an SM's four
// instructions a cycle 2.6 are issued, over half of them for integer work), so that the
// memory is not quite full: 200003 keys, 32 heads of 128 on 8 key heads, in 71.3 us (5.7
// TB/s; without the rings 94 us); 48 streams of 2000 to 8192 keys, one token each, 110 us
// (4.7 TB/s: lengths and waves are uneven). 16-bit rows: 16 streams of up to 1370 keys, 16
// heads of 64, 15.1 us (4.6 TB/s). 1370 keys of one stream, 7.2 us: launch, a chain of four
// dependent loads, and the join.
#include <algorithm>

#include "attention_rows.cuh"

namespace dav2cuda {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
// m is raised when a score exceeds it by this: p times a scale's f < 2 and 2^7 stays in f16
template <bool kS8>
constexpr float kRaise = kS8 ? 7.0f : 8.0f;
// Where m starts: finite, so that -inf - m is -inf and rows that see nothing get p = 0
// without a test; any finite score above it raises it.
constexpr float kLowest = -3.402823466e38f;

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

__device__ __forceinline__ uint32_t word(const uint4& x, int i) {
    return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w;
}

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

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16u : 0u) : "memory");
}

__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

__device__ __forceinline__ uint4 read16(uint32_t from) {
    uint4 x;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(from) : "memory");
    return x;
}

__device__ __forceinline__ uint2 read8(uint32_t from) {
    uint2 x;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(from) : "memory");
    return x;
}

// A warp's ring of 16-key tiles of K and V in shared memory, filled by asynchronous
// 16-byte copies that the warp issues for itself: no other warp waits on it. Rows
// are D values long; chunk c (16 bytes) of row r lies in 128-byte line (r C + c) / 8
// at slot (r C + c) % 8 ^ s(r), C = chunks of a row. The swizzles s make the
// copies (a row's chunks) and the fragment loads (below) free of bank conflicts:
// K: eight lanes read four chunks of rows r, r + 1; V: two chunks (of pairs
// of lanes) of rows i, 4 + i, 8 + i, 12 + i.
template <int D, bool kS8, bool kFull>
struct Ring {
    static constexpr uint32_t kTiles = kS8 || D == 64 ? 2 : 1;     // tiles of a step
    static constexpr uint32_t kChunk = 16 * kTiles;                // keys of a step
    static constexpr uint32_t kSteps = kS8 ? 2 : 3;                // steps in the ring
    static constexpr uint32_t kC = D * (kS8 ? 1 : 2) / 16;         // chunks of a row
    static constexpr uint32_t kOperand = 16 * kC * 16;             // bytes of a tile of K or V
    static constexpr uint32_t kStep = kTiles * 2 * kOperand;       // K tiles, then V tiles
    static constexpr uint32_t kBytes = kSteps * (kStep + (kS8 ? 16 : 0));  // of a warp

    static __device__ __forceinline__ uint32_t place_k(uint32_t row, uint32_t chunk) {
        const uint32_t x = row * kC + chunk;
        return kC == 4 ? x * 16 : (x ^ ((row & 1) << 2)) * 16;
    }
    static __device__ __forceinline__ uint32_t place_v(uint32_t row, uint32_t chunk) {
        const uint32_t x = row * kC + chunk, q = (row >> 2) & 3;
        return (x ^ (kC == 16 ? (q & 1) | ((q >> 1) << 2) : q << 1)) * 16;
    }

    const RowsParams& p;
    uint32_t base, scales;  // shared memory of this warp
    uint32_t seq, kv_head, len, lane;
    const uint32_t d;
    int32_t page_next[kTiles];  // pages of the step to be issued next (codes), fetched a step ahead

    __device__ Ring(const RowsParams& p, uint8_t* smem, uint32_t seq, uint32_t kv_head, uint32_t len)
        : p(p), seq(seq), kv_head(kv_head), len(len), lane(threadIdx.x & 31), d(kFull ? D : p.head_dim) {
        const uint32_t warp = threadIdx.x >> 5;
        base = smem_addr(smem) + warp * (kSteps * kStep);
        scales = smem_addr(smem) + kWarps * kSteps * kStep + warp * (kSteps * 16);
    }

    __device__ __forceinline__ void fetch_pages(uint32_t key0) {
        if constexpr (kS8) {
#pragma unroll
            for (uint32_t b = 0; b < kTiles; ++b) {
                const uint32_t key = key0 + 16 * b;
                page_next[b] =
                    key < len ? p.page_table[(uint64_t)seq * p.table_stride + (key >> p.page_shift)] : -1;
            }
        }
    }

    // Copies of the step's keys, one group whether or not there is anything to copy.
    __device__ __forceinline__ void issue(uint32_t key0, uint32_t step, bool live) {
        if (live) {
            const uint32_t to = base + step * kStep, chunks = d * (kS8 ? 1 : 2) / 16;
#pragma unroll
            for (uint32_t b = 0; b < kTiles; ++b) {
                const uint32_t key = key0 + 16 * b;
                const uint8_t *k, *v;
                uint64_t k_row, v_row;  // bytes from row to row
                bool good = true;
                if constexpr (kS8) {
                    const int32_t page = page_next[b];
                    good = page >= 0 && (uint32_t)page < p.pages;
                    if (!good && key < len && lane == 0) atomicExch(p.err, 3);
                    const uint64_t unit = (uint64_t)(uint32_t)(good ? page : 0) * p.kv_heads + kv_head;
                    const uint64_t at = ((unit << p.page_shift) + (key & ((1u << p.page_shift) - 1))) * d;
                    k = static_cast<const uint8_t*>(p.k) + at, v = static_cast<const uint8_t*>(p.v) + at;
                    k_row = v_row = d;
                    // scales; -1 and 0: no page of the cache, its keys are left out
                    const uint32_t slot = scales + step * 16 + (lane & 1) * 4 * kTiles + 4 * b;
                    if (lane < 2) {
                        if (good) copy4(slot, (lane ? p.v_scales : p.k_scales) + unit);
                        else asm volatile("st.shared.f32 [%0], %1;" ::"r"(slot), "f"(lane ? 0.0f : -1.0f) : "memory");
                    }
                } else {
                    k = static_cast<const uint8_t*>(p.k) + 2 * (seq * p.k_batch + (uint64_t)kv_head * d + key * p.k_stride);
                    v = static_cast<const uint8_t*>(p.v) + 2 * (seq * p.v_batch + (uint64_t)kv_head * d + key * p.v_stride);
                    k_row = 2 * p.k_stride, v_row = 2 * p.v_stride;
                }
#pragma unroll
                for (uint32_t i = 0; i < kC / 2; ++i) {
                    const uint32_t x = i * 32 + lane, row = x / kC, chunk = x % kC;
                    const uint32_t to_k = to + b * kOperand + place_k(row, chunk);
                    const uint32_t to_v = to + (kTiles + b) * kOperand + place_v(row, chunk);
                    if constexpr (kS8 && kFull) {  // the tile's 16 rows are consecutive
                        copy16(to_k, k + x * 16, good);
                        copy16(to_v, v + x * 16, good);
                    } else {
                        // past the end zeros: there may be no memory, or NaN
                        const bool read = good && (kFull || chunk < chunks) && (kS8 || key + row < len);
                        copy16(to_k, read ? k + row * k_row + chunk * 16 : p.k, read);
                        copy16(to_v, read ? v + row * v_row + chunk * 16 : p.v, read);
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // The oldest of kSteps - 1 groups has landed, for all lanes; all have left the step before.
    __device__ __forceinline__ void wait() const {
        asm volatile("cp.async.wait_group %0;" ::"n"(kSteps - 2) : "memory");
        __syncwarp();
    }
};

// kBF16: type of the second product's operands (false for codes).
template <int D, int NT, bool kS8, bool kBF16, bool kFull>
__global__ void __launch_bounds__(kThreads) attention_rows_kernel(const RowsParams p) {
    using Keys = Ring<D, kS8, kFull>;
    constexpr int kSteps = D / 16, kTiles = Keys::kTiles;
    constexpr uint32_t kChunk = Keys::kChunk;
    constexpr int R = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    // the rings' memory takes the warps' results at the end
    auto s_o = reinterpret_cast<float (*)[R][D + 4]>(smem);
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
    Keys f(p, smem, where.seq, kv_head, len);
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
            // exponents that would leave f32's range, stay near 1. Beside an infinity all finite
            // values stay finite
            int e = most > 0.0f ? 141 - (int)(__float_as_uint(most) >> 23) : 0;
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

    float o[kSteps][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
        m[n][0] = m[n][1] = kLowest;
        l[n][0] = l[n][1] = 0.0f;
    }

    // fragment addresses: K rows g and g + 8 of S^T (keys 4 (g / 2) + g % 2 and the
    // second next), V keys 4t .. 4t + 3
    const uint32_t kr = 4 * (g >> 1) + (g & 1);
    uint32_t step = 0, step_in = 0;
#pragma unroll
    for (uint32_t i = 0; i + 1 < Keys::kSteps; ++i) {
        const uint32_t ci = c + i * key_warps;
        f.issue(ci * kChunk, step_in++, ci < last);
        f.fetch_pages((ci + key_warps) * kChunk);
    }
    for (; c < last; c += key_warps) {
        const uint32_t key0 = c * kChunk;
        f.wait();
        {
            const uint32_t ci = c + (Keys::kSteps - 1) * key_warps;
            f.issue(ci * kChunk, step_in, ci < last);
            f.fetch_pages((ci + key_warps) * kChunk);
            step_in = step_in + 1 == Keys::kSteps ? 0 : step_in + 1;
        }
        const uint32_t from = f.base + step * Keys::kStep;
        float sk[kTiles], shift[kTiles], weight[kTiles], back_v[kTiles];  // V scale: 2^shift, f times 2^7, 2^-shift
        bool any_dead = false;
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
            sk[b] = 1.0f;
            if constexpr (kS8) {
                float sv;
                const uint32_t at = f.scales + step * 16 + 4 * b;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(sk[b]) : "r"(at) : "memory");
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(sv) : "r"(at + 4 * kTiles) : "memory");
                any_dead |= sk[b] < 0.0f;
                split_scale(sv, shift[b], weight[b], back_v[b]);
                weight[b] *= 128.0f;
            }
        }
        step = step + 1 == Keys::kSteps ? 0 : step + 1;
        float sc[kTiles][NT][4];
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
            const uint32_t k = from + b * Keys::kOperand;
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[b][n][0] = sc[b][n][1] = sc[b][n][2] = sc[b][n][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < (int)Keys::kC / 4; ++i) {
                const uint4 x4 = read16(k + Keys::place_k(kr, 4 * i + t)), y4 = read16(k + Keys::place_k(kr + 2, 4 * i + t));
                if constexpr (kS8) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t x = word(x4, j) ^ 0x80808080u, y = word(y4, j) ^ 0x80808080u;
                        const uint32_t a0 = codes_lo(x), a1 = codes_lo(y), a2 = codes_hi(x), a3 = codes_hi(y);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma_16816<false>(sc[b][n], a0, a1, a2, a3, qf[n][4 * i + j][0], qf[n][4 * i + j][1]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma_16816<kBF16>(sc[b][n], word(x4, 2 * j), word(y4, 2 * j), word(x4, 2 * j + 1),
                                             word(y4, 2 * j + 1), qf[n][2 * i + j][0], qf[n][2 * i + j][1]);
                }
            }
        }
        // scores in units of log2, the keys out of reach at -inf
        bool raise = false;
#pragma unroll
        for (int b = 0; b < kTiles; ++b)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (kS8) sc[b][n][e] = fmaf(sc[b][n][e], factor[n][e & 1] * sk[b], shift[b]);
                    else sc[b][n][e] *= factor[n][e & 1];
                }
        if (key0 + kChunk > low || any_dead) {
            const uint32_t key = key0 + 4 * (g >> 1) + (g & 1);
#pragma unroll
            for (int b = 0; b < kTiles; ++b)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (sk[b] < 0.0f || key + 16 * b + (e >= 2 ? 2 : 0) >= reach[n][e & 1]) sc[b][n][e] = -INFINITY;
        }
        float top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[n][e] = fmaxf(sc[0][n][e], sc[0][n][e + 2]);
                if (kTiles == 2) top[n][e] = fmaxf(top[n][e], fmaxf(sc[kTiles - 1][n][e], sc[kTiles - 1][n][e + 2]));
                raise |= top[n][e] > m[n][e] + kRaise<kS8>;
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = top[n][e];
#pragma unroll
                    for (int k = 4; k < 32; k *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, k));
                    x = fmaxf(x, m[n][e]);
                    const float down = ex2_approx(m[n][e] - x);
                    m[n][e] = x;
                    l[n][e] *= down;
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) o[i][n][e] *= down, o[i][n][e + 2] *= down;
                }
        }
        uint32_t pf[kTiles][NT][2];
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
            const float w = kS8 ? weight[b] : kBF16 ? 1.0f : 128.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float e4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) e4[e] = ex2_approx(sc[b][n][e] - m[n][e & 1]);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if constexpr (kS8) l[n][e] = fmaf(e4[e] + e4[e + 2], back_v[b], l[n][e]);
                    else l[n][e] += e4[e] + e4[e + 2];
                }
                pf[b][n][0] = transpose8x8(pack2<kBF16>(e4[0] * w, e4[1] * w));
                pf[b][n][1] = transpose8x8(pack2<kBF16>(e4[2] * w, e4[3] * w));
            }
        }
#pragma unroll
        for (int b = 0; b < kTiles; ++b) {
            const uint32_t from_v = from + (kTiles + b) * Keys::kOperand;
            constexpr int kV = D * (kS8 ? 1 : 2) / 32;  // words of a lane's part of a V row
            uint32_t v[4][kV];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (kV == 2) {
                    const uint2 x = read8(from_v + Keys::place_v(4 * t + i, g >> 1) + 8 * (g & 1));
                    v[i][0] = x.x, v[i][1] = x.y;
                } else {
#pragma unroll
                    for (int j = 0; j < kV; j += 4) {
                        const uint4 x = read16(from_v + Keys::place_v(4 * t + i, kV / 4 * g + j / 4));
                        v[i][j] = x.x, v[i][j + 1] = x.y, v[i][j + 2] = x.z, v[i][j + 3] = x.w;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                if constexpr (kS8) {
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
                } else {
                    const uint32_t a0 = prmt(v[0][i], v[1][i], 0x5410), a1 = prmt(v[0][i], v[1][i], 0x7632);
                    const uint32_t a2 = prmt(v[2][i], v[3][i], 0x5410), a3 = prmt(v[2][i], v[3][i], 0x7632);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816<kBF16>(o[i][n], a0, a1, a2, a3, pf[b][n][0], pf[b][n][1]);
                }
            }
        }
    }
    // the copies still under way are empty or will not be read, but they write to the rings
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();

    // this warp's result: sums over the lanes that share a column, O in true units
    const float unit = kBF16 ? 1.0f : 1.0f / 128.0f;
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

    // the join may be launched; it waits for this grid's end before it reads
    if (p.splits > 1 && !p.clusters) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // merge the key warps of each row tile: a thread takes two dims of a row
    for (uint32_t i = threadIdx.x; i < tile_rows * (D / 2); i += kThreads) {
        const uint32_t r = i / (D / 2), dim = 2 * (i - r * (D / 2));
        const uint32_t w0 = r / R * key_warps, col = r % R, row = where.tile * tile_rows + r;
        if (row >= rows || dim >= d) continue;
        float top = kLowest;
        for (uint32_t k = 0; k < key_warps; ++k) top = fmaxf(top, s_m[w0 + k][col]);
        float sum = 0.0f, x[2] = {0.0f, 0.0f};
        for (uint32_t k = 0; k < key_warps; ++k) {
            const float a = ex2_approx(s_m[w0 + k][col] - top);
            sum += a * s_l[w0 + k][col];
            const float2 b = *reinterpret_cast<const float2*>(&s_o[w0 + k][col][dim]);
            x[0] += a * b.x;
            x[1] += a * b.y;
        }
        if (p.splits == 1) {
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
            x[0] *= inv, x[1] *= inv;
            store_out(p, row_at(p, where, kv_head, row, p.out_batch, p.out_stride) + dim, x, 2);
        } else if (p.clusters) {
            *reinterpret_cast<float2*>(&s_o[w0][col][dim]) = make_float2(x[0], x[1]);  // read by this thread alone
            if (dim == 0) c_m[r] = top, c_l[r] = sum;
        } else {
            const uint64_t slot = part_at(p, where, kv_head, row, blockIdx.z);
            if (dim == 0) p.part_ml[slot] = make_float2(top, sum);
            if (sum != 0.0f) *reinterpret_cast<float2*>(p.part_o + slot * d + dim) = make_float2(x[0], x[1]);
        }
    }
    if (!p.clusters) return;
    // the splits are a cluster: each block merges its share of the rows' dims
    cluster_sync();
    for (uint32_t i = blockIdx.z * kThreads + threadIdx.x; i < tile_rows * (D / 2); i += p.splits * kThreads) {
        const uint32_t r = i / (D / 2), dim = 2 * (i - r * (D / 2));
        const uint32_t w0 = r / R * key_warps, col = r % R, row = where.tile * tile_rows + r;
        if (row >= rows || dim >= d) continue;
        float top = kLowest;
        for (uint32_t k = 0; k < p.splits; ++k) top = fmaxf(top, cluster_load(cluster_place(&c_m[r], k)));
        float sum = 0.0f, x[2] = {0.0f, 0.0f};
        for (uint32_t k = 0; k < p.splits; ++k) {
            const float a = ex2_approx(cluster_load(cluster_place(&c_m[r], k)) - top);
            sum += a * cluster_load(cluster_place(&c_l[r], k));
            const float2 b = cluster_load2(cluster_place(&s_o[w0][col][dim], k));
            x[0] += a * b.x;
            x[1] += a * b.y;
        }
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        x[0] *= inv, x[1] *= inv;
        store_out(p, row_at(p, where, kv_head, row, p.out_batch, p.out_stride) + dim, x, 2);
    }
    cluster_sync();  // no block leaves while another reads its shared memory
}

// Joins the splits of a row, four dims to a lane: a warp to a row or (kWide, many splits)
// a block, each warp every fourth split and then the warps' sums. Launched while the
// kernel of the splits still runs; waits for its end.
template <bool kWide>
__global__ void __launch_bounds__(kThreads) attention_join_kernel(const RowsParams p, const uint64_t rows) {
    __shared__ float s_f[kWide ? kMaxSplits : 1];
    __shared__ float4 s_x[kWide ? kWarps : 1][32];
    constexpr uint32_t kLoads = kWide ? kMaxSplits / 32 : 1;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t row = kWide ? (uint64_t)blockIdx.x : (uint64_t)blockIdx.x * kWarps + warp;
    const uint32_t heads = p.kv_heads * p.group;
    const uint64_t token = row / heads;
    const uint32_t head = (uint32_t)(row - token * heads);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // rows of no sequence stay as they were
    if (row >= rows || (p.query_begin && ((int64_t)token < p.query_begin[0] || (int64_t)token >= p.query_begin[p.sequences])))
        return;
    float top = kLowest, sum = 0.0f, weight = 0.0f;
    float2 ml[kLoads];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
        const uint32_t k = 32 * i + lane;
        ml[i] = k < p.splits ? p.part_ml[row * p.splits + k] : make_float2(kLowest, 0.0f);
        top = fmaxf(top, ml[i].x);
    }
    top = warp_max(top);
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
        // a split with no key in reach has written no sums
        weight = ml[i].y != 0.0f ? ex2_approx(ml[i].x - top) : 0.0f;
        sum += weight * ml[i].y;
        if (kWide && warp == 0) s_f[32 * i + lane] = weight;
    }
    sum = warp_sum(sum);
    const uint32_t dim = 4 * lane;
    const float* from = p.part_o + row * p.splits * p.head_dim + dim;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if constexpr (kWide) {
        __syncthreads();
        if (dim < p.head_dim) {
#pragma unroll 8
            for (uint32_t k = warp; k < p.splits; k += kWarps) {
                const float f = s_f[k];
                if (f == 0.0f) continue;
                const float4 o = *reinterpret_cast<const float4*>(from + (uint64_t)k * p.head_dim);
                x.x += f * o.x, x.y += f * o.y, x.z += f * o.z, x.w += f * o.w;
            }
        }
        s_x[warp][lane] = x;
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (uint32_t w = 1; w < kWarps; ++w) {
            const float4 y = s_x[w][lane];
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        }
    } else {
#pragma unroll 8
        for (uint32_t k = 0; k < p.splits; ++k) {
            const float f = __shfl_sync(0xffffffffu, weight, k);
            if (f == 0.0f || dim >= p.head_dim) continue;
            const float4 o = *reinterpret_cast<const float4*>(from + (uint64_t)k * p.head_dim);
            x.x += f * o.x, x.y += f * o.y, x.z += f * o.z, x.w += f * o.w;
        }
    }
    if (dim >= p.head_dim) return;
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    const float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    const uint64_t batch = p.query_begin ? 0 : token / p.queries;
    const uint64_t at = p.query_begin ? token * p.out_stride
                                      : batch * p.out_batch + (token - batch * p.queries) * p.out_stride;
    store_out(p, at + (uint64_t)head * p.head_dim + dim, y, 4);
}

template <int D, int NT, bool kS8, bool kBF16, bool kFull>
int start(const RowsParams& p, uint32_t slots, cudaStream_t st) {
    cudaLaunchAttribute cluster[1];
    cluster[0].id = cudaLaunchAttributeClusterDimension;
    cluster[0].val.clusterDim.x = 1, cluster[0].val.clusterDim.y = 1, cluster[0].val.clusterDim.z = p.splits;
    constexpr uint32_t kSmem = std::max<uint32_t>(kWarps * Ring<D, kS8, kFull>::kBytes, kWarps * 8 * NT * (D + 4) * 4);
    auto kernel = attention_rows_kernel<D, NT, kS8, kBF16, kFull>;
    static std::atomic<uint64_t> configured;  // one bit per device ordinal
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured_on(configured, dev)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem) != cudaSuccess ||
            cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 (int)cudaSharedmemCarveoutMaxShared) != cudaSuccess)
            return set_error(DAV2CUDA_LAUNCH_FAILED, "attention: cannot set shared memory size");
        mark_configured(configured, dev);
    }
    cudaLaunchConfig_t config{};
    config.dynamicSmemBytes = kSmem;
    config.gridDim = dim3(slots, p.kv_heads, p.splits);
    config.blockDim = dim3(kThreads);
    config.stream = st;
    config.attrs = cluster;
    config.numAttrs = p.clusters ? 1 : 0;
    cudaLaunchKernelEx(&config, kernel, p);
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
    cudaLaunchAttribute early[1];
    early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    const bool wide = p.splits > 32;
    config.gridDim = dim3((uint32_t)(wide ? rows : (rows + kWarps - 1) / kWarps));
    config.blockDim = dim3(kThreads);
    config.stream = st;
    config.attrs = early;
    config.numAttrs = 1;
    cudaLaunchKernelEx(&config, wide ? attention_join_kernel<true> : attention_join_kernel<false>, p, rows);
    return check_launch("attention_join");
}

}  // namespace dav2cuda

// Attention of many query rows on tcgen05 tensor cores, for the two sources of
// keys and values of attention_rows.cu (16-bit rows, pages of int8 codes).
//
// A block takes two tiles of 128 rows (query x head of the group that shares a key
// head) and walks the keys in blocks of 128:
//   S_t = Q_t K^T (128 x 128, f32 in tensor memory), P_t = 2^(S_t - m) in 16 bits,
//   O_t += P_t V (128 x D, f32 in tensor memory), l_t += sum P_t
// One thread owns one row: it loads its 128 scores, takes the maximum, exponentiates
// and writes P into tensor memory, from where the second product reads it as its A
// operand, so that P never passes through shared memory. m follows the row's maximum
// only when that exceeds it by 8 (log2 units), and then the thread rescales its row
// of O; S_t's barrier tells that the previous P V is done, since it was issued before.
// While one tile's softmax runs, the tensor cores work on the other tile.
//
//   warps 0-3, 4-7   softmax of tile 0, 1 (and, first, their rows of Q to shared memory)
//   warp 8           products: P_0 V_j, S_0 of j + 1, P_1 V_j, S_1 of j + 1
//   warp 9           16-bit rows: TMA of K_j, V_j into a ring of 128-key tiles
//   warps 9-11       codes: int8 from the pages into the same tiles as f16
// The 128-byte-swizzled tiles are 64 dims wide; heads above 64 take two of them.
//
// Keys past the end: scores are replaced by -inf; the rows of V behind the last
// key are set to zero in shared memory before the last product, as they may hold
// NaN. Codes: K's scale multiplies the scores of its page's keys, V's scale, over
// the largest of the sequence, multiplies P before it is rounded.
// Every wait is bounded (kWaitTimeoutNs); a timeout sets the device error word.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "abi_check.h"
#include "attention_rows.cuh"

namespace dav2cuda {
namespace {

constexpr uint32_t kTileRows = 128;
constexpr uint32_t kKeys = 128;        // keys of a block
constexpr uint32_t kAtom = 128 * 128;  // bytes of 128 rows x 64 dims of 16 bits
constexpr float kRaise = 8.0f;
constexpr uint32_t kSoftmaxThreads = 256;
constexpr uint32_t kConverters = 3;    // 12 warps in all: 168 registers a thread

template <int D, bool kS8>
struct Layout {
    static constexpr uint32_t kOperand = D / 64 * kAtom;   // bytes of 128 rows
    static constexpr uint32_t kStages = D == 64 ? 8 : 5;   // K or V tiles in flight
    static constexpr uint32_t kThreads = kSoftmaxThreads + (kS8 ? 1 + kConverters : 2) * 32;
    static constexpr uint32_t kSmem = (2 + kStages) * kOperand + 1024;
    // S_0, S_1, then O_0, O_1; P shares S's columns
    static constexpr uint32_t kO = 256;
};

__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 8-column TMEM row access (the rare O rescale; keeps register use low)
__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// MN-major operand (V: keys x dims, dims contiguous), 128-byte swizzle: 8-key
// groups 1024 B apart, 64-dim groups one atom apart.
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(kAtom >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
           (static_cast<uint64_t>(2) << 61);
}

// Byte of (row, 8-dim chunk) in a swizzled operand.
__device__ __forceinline__ uint32_t chunk_at(uint32_t row, uint32_t chunk) {
    return (chunk >> 3) * kAtom + row * 128u + (((chunk & 7u) ^ (row & 7u)) << 4);
}

template <int D, bool kS8, bool kBF16>
__global__ void __launch_bounds__((Layout<D, kS8>::kThreads), 1)
    attention_tiles_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                           const RowsParams p) {
    using L = Layout<D, kS8>;
    constexpr uint32_t kStages = L::kStages;
    extern __shared__ uint8_t smem[];
    uint8_t* sQ = smem;                        // [tile]
    uint8_t* sKV = smem + 2 * L::kOperand;     // [stage]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + kStages * L::kOperand);
    uint64_t* full = bars;               // [stage]
    uint64_t* empty = full + kStages;    // [stage]
    uint64_t* q_full = empty + kStages;  // [tile]
    uint64_t* s_full = q_full + 2;       // [tile]
    uint64_t* p_full = s_full + 2;       // [tile]
    uint64_t* o_full = p_full + 2;
    uint64_t* drain = o_full + 1;
    float* s_top = reinterpret_cast<float*>(drain + 1);            // [warp]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_top + 16);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    RowTile where;
    if (!find_row_tile(where, p, blockIdx.x, 2 * kTileRows)) return;
    const uint32_t kv_head = blockIdx.y;
    const uint32_t len = keys_of(p, where.seq);
    const uint32_t row0 = where.tile * 2 * kTileRows;
    const uint32_t tiles = where.rows - row0 > kTileRows ? 2u : 1u;
    // the key blocks of this split, up to the last row's reach
    const uint32_t reach_top = reach_of(p, where, len, min(where.rows, row0 + 2 * kTileRows) - 1);
    const uint32_t all = (len + kKeys - 1) / kKeys, per_split = (all + p.splits - 1) / p.splits;
    const uint32_t first = blockIdx.z * per_split;
    const uint32_t last = min(min(all, first + per_split), (reach_top + kKeys - 1) / kKeys);
    const uint32_t blocks = last > first ? last - first : 0;

    if ((smem_addr(smem) & 1023u) != 0) {  // the 128-byte swizzle needs 1 KB aligned tiles
        if (threadIdx.x == 0) atomicExch(p.err, 2);
        return;
    }
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kStages; ++i) {
            mbar_init(&full[i], kS8 ? kConverters : 1);
            mbar_init(&empty[i], 1);
        }
        for (uint32_t t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 4);
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 4);
        }
        mbar_init(o_full, 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
        if (!kS8) {
            tma_prefetch_desc(&tm_k);
            tma_prefetch_desc(&tm_v);
        }
    }
    if (warp == 8) tmem_alloc(tmem_slot, 512);
    float v_top = 1.0f;
    if constexpr (kS8) {
        // the largest V scale of the keys in reach
        float top = 0.0f;
        const uint32_t page_end = (min(len, last * kKeys) + (1u << p.page_shift) - 1) >> p.page_shift;
        for (uint32_t i = ((first * kKeys) >> p.page_shift) + threadIdx.x; i < page_end; i += L::kThreads) {
            const int32_t page = p.page_table[(uint64_t)where.seq * p.table_stride + i];
            if (page >= 0 && (uint32_t)page < p.pages)
                top = fmaxf(top, p.v_scales[(uint64_t)page * p.kv_heads + kv_head]);
        }
        top = warp_max(top);
        if (lane == 0) s_top[warp] = top;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if constexpr (kS8) {
        float top = 1e-30f;
        for (uint32_t i = 0; i < L::kThreads / 32; ++i) top = fmaxf(top, s_top[i]);
        v_top = top;
    }
    bool mma_issued = false;

    if (warp < 8) {
        // ------------------------------------------------------------ softmax
        const uint32_t t = warp >> 2, quarter = warp & 3u;
        const uint32_t r = quarter * 32u + lane;                      // row of the tile
        const uint32_t row = row0 + t * kTileRows + r;                // row of the sequence
        const uint32_t tS = tmem + t * 128u + ((quarter * 32u) << 16);
        const uint32_t tO = tmem + L::kO + t * D + ((quarter * 32u) << 16);
        const bool live = row < where.rows;
        if (t < tiles && blocks) {
            // this row of Q; a negative scale goes into its sign. For codes it is
            // brought into f16's range by a power of two.
            const uint16_t* q = static_cast<const uint16_t*>(p.q) +
                                (live ? row_at(p, where, kv_head, row, p.q_batch, p.q_stride) : 0);
            uint4 x[D / 8];
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                x[i] = live && 8 * i < p.head_dim ? *reinterpret_cast<const uint4*>(q + 8 * i) : make_uint4(0, 0, 0, 0);
            const uint32_t sign = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
            float c = fabsf(p.scale_log2);
            if constexpr (kS8) {
                float most = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const uint32_t w4[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 a = unpack2(w4[e], p.q_bf16);
                        most = fmax3(most, fabsf(a.x), fabsf(a.y));
                    }
                }
                int e = most > 0.0f && most < INFINITY ? 141 - (int)(__float_as_uint(most) >> 23) : 0;
                e = max(-120, min(120, e));
                const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                c *= __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    uint32_t* w4 = reinterpret_cast<uint32_t*>(&x[i]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2 a = unpack2(w4[k], p.q_bf16);
                        w4[k] = pack2<false>(a.x * up, a.y * up);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<uint4*>(sQ + t * L::kOperand + chunk_at(r, i)) =
                    make_uint4(x[i].x ^ sign, x[i].y ^ sign, x[i].z ^ sign, x[i].w ^ sign);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[t]);

            const uint32_t reach = reach_of(p, where, len, row);
            const uint32_t low = __reduce_min_sync(0xffffffffu, live ? reach : 0xFFFFFFFFu);
            auto warp_wait = [&](uint64_t* bar, uint32_t parity) -> bool {
                return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.err));
            };
            // codes: lane i has the K scale (i < 8), lane 8 + i the V scale over the largest,
            // of the block's keys 16i .. 16i + 15; fetched a block ahead. -1: no such page
            auto scale_of = [&](uint32_t j) -> float {
                const uint32_t key = (first + j) * kKeys + 16u * (lane & 7u);
                if (lane >= 16 || key >= len) return 0.0f;
                const int32_t page = p.page_table[(uint64_t)where.seq * p.table_stride + (key >> p.page_shift)];
                if (page < 0 || (uint32_t)page >= p.pages) return lane < 8 ? -1.0f : 0.0f;
                const uint64_t unit = (uint64_t)page * p.kv_heads + kv_head;
                return lane < 8 ? p.k_scales[unit] : p.v_scales[unit] * (128.0f / v_top);
            };
            float scale_next = 0.0f, scale_now = 0.0f;
            if constexpr (kS8) scale_next = scale_of(0);
            float m = -INFINITY, l = 0.0f;
            // f16: P is kept times 2^7, which leaves f16 down to 2^-31 of the row's largest
            constexpr float kShift = kBF16 || kS8 ? 0.0f : 7.0f;
            bool ok = true;
            for (uint32_t j = 0; j < blocks; ++j) {
                if (!warp_wait(&s_full[t], j & 1u)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint32_t sr[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(tS + 32u * i, sr[i]);
                tmem_ld_wait();
                float s[128];
#pragma unroll
                for (int i = 0; i < 128; ++i) s[i] = __uint_as_float(sr[i >> 5][i & 31]);
                const uint32_t key0 = (first + j) * kKeys;
                if constexpr (kS8) {
                    scale_now = scale_next;
                    if (j + 1 < blocks) scale_next = scale_of(j + 1);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float f = __shfl_sync(0xffffffffu, scale_now, i) * c;
#pragma unroll
                        for (int e = 0; e < 16; ++e) s[16 * i + e] = f >= 0.0f ? s[16 * i + e] * f : -INFINITY;
                    }
                }
                if (key0 + kKeys > low) {
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (key0 + i >= reach) s[i] = -INFINITY;
                }
                float a[43];
#pragma unroll
                for (int i = 0; i < 42; ++i) a[i] = fmax3(s[3 * i], s[3 * i + 1], s[3 * i + 2]);
                a[42] = fmaxf(s[126], s[127]);
#pragma unroll
                for (int i = 0; i < 14; ++i) a[i] = fmax3(a[3 * i], a[3 * i + 1], a[3 * i + 2]);
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = fmax3(a[3 * i], a[3 * i + 1], a[3 * i + 2]);
                float top = fmax3(fmax3(a[0], a[1], a[2]), fmax3(a[3], a[12], a[13]), a[42]);
                if constexpr (!kS8) top = top == -INFINITY ? top : top * c;
                const bool raise = top > m + kRaise;
                if (__any_sync(0xffffffffu, raise)) {
                    const float up = fmaxf(m, top);
                    const float down = up == -INFINITY ? 1.0f : ex2_approx(m - up);
                    if (j > 0) {  // O holds the blocks before: P V was issued before S
#pragma unroll 1
                        for (uint32_t k = 0; k < D / 8; ++k) {
                            uint32_t o[8];
                            tmem_ld_x8(tO + 8u * k, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * down);
                            tmem_st_x8(tO + 8u * k, o);
                        }
                        tmem_st_wait();
                    }
                    l *= down;
                    m = up;
                }
                const float off = kShift - (m == -INFINITY ? 0.0f : m);
                float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[32];
                    float sv[4] = {1.0f, 1.0f, 1.0f, 1.0f};
                    if constexpr (kS8) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) sv[i] = __shfl_sync(0xffffffffu, scale_now, 8 + 4 * h + i);
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float x = s[64 * h + 2 * i], y = s[64 * h + 2 * i + 1];
                        if constexpr (kS8) {
                            x = ex2_approx(x + off), y = ex2_approx(y + off);
                            ls[(2 * i) & 3] += x, ls[(2 * i + 1) & 3] += y;
                            const float f = sv[i / 8];
                            w[i] = pack2<false>(x * f, y * f);
                        } else {
                            f2_fma(x, y, x, y, c, c, off, off);
                            x = ex2_approx(x), y = ex2_approx(y);
                            f2_add(ls[(2 * i) & 3], ls[(2 * i + 1) & 3], ls[(2 * i) & 3], ls[(2 * i + 1) & 3], x, y);
                            w[i] = pack2<kBF16>(x, y);
                        }
                    }
                    tmem_st_32x32b_x32(tS + 32u * h, w);
                }
                l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            if (p.splits > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            if (ok) ok = warp_wait(o_full, 0);
            tc_fence_after();
            if (ok) {
                const float unit = kS8 ? v_top * (1.0f / 128.0f) : 1.0f;
                const float back = kShift != 0.0f ? 1.0f / 128.0f : 1.0f;
                const float f = p.splits == 1 ? (l > 0.0f ? unit / l : 0.0f) : unit * back;
                const uint64_t slot = live && p.splits > 1 ? part_at(p, where, kv_head, row, blockIdx.z) : 0;
                const uint64_t at = live ? row_at(p, where, kv_head, row, p.out_batch, p.out_stride) : 0;
                if (live && p.splits > 1) p.part_ml[slot] = make_float2(m, l * back);
#pragma unroll 1
                for (uint32_t k = 0; k < D / 32; ++k) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(tO + 32u * k, o);
                    tmem_ld_wait();
                    if (!live) continue;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        if (32 * k + i >= p.head_dim) continue;
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = l > 0.0f ? __uint_as_float(o[i + e]) * f : 0.0f;
                        if (p.splits > 1) {
                            float4* to = reinterpret_cast<float4*>(p.part_o + slot * p.head_dim + 32 * k + i);
                            to[0] = make_float4(x[0], x[1], x[2], x[3]);
                            to[1] = make_float4(x[4], x[5], x[6], x[7]);
                        } else if (p.out_kind == 0) {
                            float4* to = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at + 32 * k + i);
                            to[0] = make_float4(x[0], x[1], x[2], x[3]);
                            to[1] = make_float4(x[4], x[5], x[6], x[7]);
                        } else {
                            uint32_t w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                w[e] = p.out_kind == 1 ? pack2<true>(x[2 * e], x[2 * e + 1])
                                                       : pack2<false>(x[2 * e], x[2 * e + 1]);
                            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at + 32 * k + i) =
                                make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
            }
        } else if (t < tiles && live) {
            // no key in reach
            if (p.splits > 1) {
                p.part_ml[part_at(p, where, kv_head, row, blockIdx.z)] = make_float2(-INFINITY, 0.0f);
            } else {
                const uint64_t at = row_at(p, where, kv_head, row, p.out_batch, p.out_stride);
                const float zero[2] = {0.0f, 0.0f};
                for (uint32_t i = 0; i < p.head_dim; i += 2) store_out(p, at + i, zero, 2);
            }
        }
    } else if (warp == 8) {
        // ----------------------------------------------------------- products
        constexpr uint32_t ab = kBF16 ? 1u : 0u;
        constexpr uint32_t idesc_s = make_idesc(1u, ab, 128u, 128u);
        constexpr uint32_t idesc_o = make_idesc(1u, ab, 128u, D) | (1u << 16);  // V is MN-major
        auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
            return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.err));
        };
        auto issue_s = [&](uint32_t t, uint32_t stage) {
            const uint32_t q = smem_addr(sQ + t * L::kOperand), k = smem_addr(sKV + stage * L::kOperand);
#pragma unroll
            for (uint32_t kk = 0; kk < D / 16; ++kk) {
                const uint32_t at = (kk / 4) * kAtom + 32u * (kk % 4);
                umma<false>(tmem + 128u * t, smem_desc_sw128(q + at), smem_desc_sw128(k + at), idesc_s, kk ? 1u : 0u);
            }
            umma_commit(&s_full[t]);
        };
        // K_j is tile 2j, V_j tile 2j + 1 of the ring
        bool ok = true;
        if (blocks) {
            for (uint32_t t = 0; t < tiles && ok; ++t) ok = wait(&q_full[t], 0);
            ok = ok && wait(&full[0], 0);
            if (ok) {
                tc_fence_after();
                if (lane == 0) {
                    for (uint32_t t = 0; t < tiles; ++t) issue_s(t, 0);
                    umma_commit(&empty[0]);
                    mma_issued = true;
                }
                __syncwarp();
            }
        }
        for (uint32_t j = 0; ok && j < blocks; ++j) {
            const uint32_t nv = 2 * j + 1, nk = 2 * j + 2;
            const uint32_t sv = nv % kStages, sk = nk % kStages;
            const bool more = j + 1 < blocks;
            const uint32_t valid = min(kKeys, len - (first + j) * kKeys);
            const uint32_t steps = (valid + 15u) / 16u;
            for (uint32_t t = 0; t < tiles && ok; ++t) {
                if (t == 0) {
                    ok = wait(&full[sv], (nv / kStages) & 1u);
                    if (ok && !kS8 && (valid & 15u)) {
                        // rows of V behind the last key, up to the product's end
                        uint8_t* v = sKV + sv * L::kOperand;
                        for (uint32_t i = lane; i < (16u - (valid & 15u)) * (D / 8); i += 32) {
                            const uint32_t row = valid + i / (D / 8);
                            *reinterpret_cast<uint4*>(v + chunk_at(row, i % (D / 8))) = make_uint4(0, 0, 0, 0);
                        }
                        fence_async_smem();
                        __syncwarp();
                    }
                }
                ok = ok && wait(&p_full[t], j & 1u);
                if (ok && more && t == 0) ok = wait(&full[sk], (nk / kStages) & 1u);
                if (!ok) break;
                tc_fence_after();
                if (lane == 0) {
                    const uint32_t v = smem_addr(sKV + sv * L::kOperand);
                    for (uint32_t kk = 0; kk < steps; ++kk)
                        umma_ts(tmem + L::kO + t * D, tmem + 128u * t + 8u * kk, desc_v(v + kk * 2048u), idesc_o,
                                (j | kk) ? 1u : 0u);
                    if (t + 1 == tiles) umma_commit(&empty[sv]);
                    if (more) {
                        issue_s(t, sk);
                        if (t + 1 == tiles) umma_commit(&empty[sk]);
                    } else if (t + 1 == tiles) {
                        umma_commit(o_full);
                    }
                }
                __syncwarp();
            }
        }
    } else if constexpr (!kS8) {
        // ---------------------------------------------------------------- TMA
        if (lane == 0) {
            const int batch = p.k_batch ? (int)where.seq : 0, v_batch = p.v_batch ? (int)where.seq : 0;
            for (uint32_t n = 0; n < 2 * blocks; ++n) {
                const uint32_t st = n % kStages;
                if (*abort_flag || !mbar_wait(&empty[st], ((n / kStages) & 1u) ^ 1u, abort_flag, p.err)) break;
                mbar_arrive_expect_tx(&full[st], L::kOperand);
                const int key0 = (int)((first + n / 2) * kKeys);
#pragma unroll
                for (int h = 0; h < D / 64; ++h)
                    tma_load_4d(sKV + st * L::kOperand + h * kAtom, n & 1 ? &tm_v : &tm_k, &full[st], 64 * h,
                                (int)kv_head, key0, n & 1 ? v_batch : batch);
            }
        }
    } else {
        // -------------------------------------------------------------- codes
        // a thread converts 16 dims of a key at a time
        constexpr uint32_t kParts = D / 16, kStep = 32 * kConverters;
        constexpr uint32_t kLoads = (kKeys * kParts + kStep - 1) / kStep;
        const uint32_t i0 = threadIdx.x - (kSoftmaxThreads + 32);
        const uint32_t in_page = (1u << p.page_shift) - 1;
        // lane i < 8 has the page of keys 16i .. 16i + 15 of a block, fetched a block ahead
        auto page_of = [&](uint32_t j) -> int32_t {
            const uint32_t key = (first + j) * kKeys + 16u * (lane & 7u);
            if (key >= len) return -1;
            const int32_t page = p.page_table[(uint64_t)where.seq * p.table_stride + (key >> p.page_shift)];
            if (page < 0 || (uint32_t)page >= p.pages) {
                atomicExch(p.err, 3);
                return -1;
            }
            return page;
        };
        int32_t page_now = -1, page_next = blocks ? page_of(0) : -1;
        uint4 x[kLoads];
        auto load = [&](uint32_t n) {
            const int8_t* codes = static_cast<const int8_t*>(n & 1 ? p.v : p.k);
            if (!(n & 1)) {
                page_now = page_next;
                if (n / 2 + 1 < blocks) page_next = page_of(n / 2 + 1);
            }
#pragma unroll
            for (uint32_t k = 0; k < kLoads; ++k) {
                const uint32_t i = i0 + kStep * k, key = i / kParts, part = i % kParts;
                const int32_t page = __shfl_sync(0xffffffffu, page_now, (key >> 4) & 7);
                x[k] = make_uint4(0, 0, 0, 0);
                if (page >= 0 && key < kKeys && 16 * part < p.head_dim)
                    x[k] = *reinterpret_cast<const uint4*>(
                        codes + ((((uint64_t)page * p.kv_heads + kv_head) << p.page_shift) +
                                 (((first + n / 2) * kKeys + key) & in_page)) * p.head_dim + 16 * part);
            }
        };
        if (blocks) load(0);
        for (uint32_t n = 0; n < 2 * blocks; ++n) {
            const uint32_t st = n % kStages;
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[st], ((n / kStages) & 1u) ^ 1u, abort_flag, p.err))) break;
            uint8_t* to = sKV + st * L::kOperand;
#pragma unroll
            for (uint32_t k = 0; k < kLoads; ++k) {
                const uint32_t i = i0 + kStep * k, key = i / kParts, part = i % kParts;
                if (key >= kKeys) continue;
                const uint32_t w4[4] = {x[k].x ^ 0x80808080u, x[k].y ^ 0x80808080u, x[k].z ^ 0x80808080u,
                                        x[k].w ^ 0x80808080u};
                *reinterpret_cast<uint4*>(to + chunk_at(key, 2 * part)) =
                    make_uint4(codes_lo(w4[0]), codes_hi(w4[0]), codes_lo(w4[1]), codes_hi(w4[1]));
                *reinterpret_cast<uint4*>(to + chunk_at(key, 2 * part + 1)) =
                    make_uint4(codes_lo(w4[2]), codes_hi(w4[2]), codes_lo(w4[3]), codes_hi(w4[3]));
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[st]);
            if (n + 1 < 2 * blocks) load(n + 1);
        }
    }

    __syncthreads();
    if (*abort_flag) {
        if (warp == 8 && lane == 0 && mma_issued) {
            umma_commit(drain);
            const unsigned long long t0 = globaltimer();
            while (!mbar_try_wait(smem_addr(drain), 0) && globaltimer() - t0 < 100000000ull) {
            }
        }
        if (threadIdx.x == 0) {  // copies in flight land before the block's memory is given back
            const unsigned long long t0 = globaltimer();
            while (globaltimer() - t0 < 2000000ull) {
            }
        }
        __syncthreads();
    }
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

// [batch][keys][kv_heads][head_dim] as boxes of 64 dims x 128 keys of one head;
// dims and keys past the end read as zero.
bool encode_keys(CUtensorMap& tm, const RowsParams& p, const void* rows, uint64_t stride, uint64_t batch_stride,
                 bool bf16) {
    const uint64_t row = (uint64_t)p.kv_heads * p.head_dim;
    const bool batches = batch_stride && p.sequences > 1;
    const cuuint64_t dims[4] = {p.head_dim, p.kv_heads, p.max_length, batches ? p.sequences : 1u};
    const cuuint64_t strides[3] = {p.head_dim * 2ull, (p.max_length > 1 ? stride : row) * 2,
                                   (batches ? batch_stride : row) * 2};
    const cuuint32_t box[4] = {64, 1, kKeys, 1}, each[4] = {1, 1, 1, 1};
    return g_encode(&tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                    const_cast<void*>(rows), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kS8, bool kBF16>
int start(const CUtensorMap& k, const CUtensorMap& v, const RowsParams& p, uint32_t slots, cudaStream_t st) {
    using L = Layout<D, kS8>;
    auto kernel = attention_tiles_kernel<D, kS8, kBF16>;
    static std::atomic<uint64_t> configured;  // one bit per device ordinal
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured_on(configured, dev)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem) != cudaSuccess ||
            cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 (int)cudaSharedmemCarveoutMaxShared) != cudaSuccess)
            return set_error(DAV2CUDA_LAUNCH_FAILED, "attention: cannot set shared memory size");
        mark_configured(configured, dev);
    }
    kernel<<<dim3(slots, p.kv_heads, p.splits), L::kThreads, L::kSmem, st>>>(k, v, p);
    return check_launch("attention_tiles");
}

}  // namespace

int launch_attention_tiles(const RowsParams& p, uint32_t slots, bool s8, bool bf16, cudaStream_t st) {
    CUtensorMap k{}, v{};
    if (!s8 && p.max_length) {
        std::call_once(g_encode_once, [] {
            void* fn = nullptr;
            cudaDriverEntryPointQueryResult q;
            if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
                q == cudaDriverEntryPointSuccess)
                g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
        });
        if (!g_encode) return set_error(DAV2CUDA_INTERNAL_ERROR, "cuTensorMapEncodeTiled unavailable");
        if (!encode_keys(k, p, p.k, p.k_stride, p.k_batch, bf16) || !encode_keys(v, p, p.v, p.v_stride, p.v_batch, bf16))
            return set_error(DAV2CUDA_INVALID_ARGUMENT, "attention: tensor map encoding failed");
    }
    const bool small = p.head_dim <= 64;
    if (s8) return small ? start<64, true, false>(k, v, p, slots, st) : start<128, true, false>(k, v, p, slots, st);
    if (bf16) return small ? start<64, false, true>(k, v, p, slots, st) : start<128, false, true>(k, v, p, slots, st);
    return small ? start<64, false, false>(k, v, p, slots, st) : start<128, false, false>(k, v, p, slots, st);
}

}  // namespace dav2cuda

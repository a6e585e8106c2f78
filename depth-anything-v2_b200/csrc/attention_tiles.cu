// Attention of many query rows on tcgen05 tensor cores, for the two sources of
// keys and values of attention_rows.cu (16-bit rows, pages of int8 codes).
//
// A unit of work is two tiles of 128 rows (query x head of the group that shares a key
// head) against the keys in blocks of 128:
//   S_t = Q_t K^T (128 x 128, f32 in tensor memory), P_t = 2^(S_t - m) in 16 bits,
//   O_t += P_t V (128 x D, f32 in tensor memory), l_t += sum P_t
// One thread owns one row: it loads its 128 scores, takes the maximum, exponentiates
// and writes P into tensor memory, from where the second product reads it as its A
// operand, so that P never passes through shared memory. m follows the row's maximum
// only when that exceeds it by 8 (log2 units), and then the thread rescales its row
// of O. While one tile's softmax runs, the tensor cores work on the other tile; at
// D = 64 also S of the next block, as P has columns of its own.
//
// One block runs on an SM at a time and takes over, unit after unit, that of a
// block that has not started yet (cluster launch control), so that units of different
// lengths spread evenly; its roles run ahead of one another across units: Q and the first
// keys of the next unit are loaded, and its first S computed, while the softmax warps
// still write the last unit's rows.
//
//   warps 0-3, 4-7   softmax of tile 0, 1
//   16-bit rows:     warps 8, 9 products of tile 0, 1; warp 10 TMA of K_j, V_j into a
//                    ring of 128-key tiles; warp 11 rows of Q (TMA where the heads of a
//                    group divide 128, else copies)
//   codes:           warp 8 products of both; warps 9-11 int8 from the pages, by bulk
//                    copies, to f16 in the same ring; the softmax warps bring Q, scaled by
//                    a power of two for each row into f16's range
// The 128-byte-swizzled tiles are 64 dims wide; heads above 64 take two of them.
//
// Keys past the end: scores are replaced by -inf; the rows of V behind the last
// key are set to zero in shared memory before the last product, as they may hold
// NaN. Codes: K's scale multiplies the scores of its page's keys; V's scale 2^e f adds
// e to them and multiplies P by f before it is rounded, and the sum takes P times 2^-e, so
// that P's range is that of what the row's keys contribute (attention_rows.cuh).
//
// No unit of the SM is full (16-bit rows: issue slots 34 to 38%, exponential unit 52%, tensor
// pipe 25% at D = 64, 52% at D = 128): the time is each tile's chain from its scores to its next
// ones (load, maximum, exponentials, store, products), hidden by the other tile's alone. For
// 128 keys the exponential units need 1.1 us at D = 64 and 128 alike, the products 0.65 and 1.1.
// Measured, bf16: 8 x 1370 x 1370, 16 heads of 64, 128 us (481 TFLOP/s); 4 x 1370 x 5477, 16
// heads of 128 on 4 key heads, padded batch, 212 us (906 TFLOP/s). Codes: the chain of one
// issuer and the conversion on top; 700 queries over 6 caches of up to 6000 tokens, 32 heads
// of 128 on 8 key heads, 134 us (297 TFLOP/s).
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
// P is at most 2^8; codes: 2^7, times f < 2 and 2^7 in f16
template <bool kS8>
constexpr float kRaise = kS8 ? 7.0f : 8.0f;
constexpr uint32_t kSoftmaxWarps = 8;
constexpr uint32_t kConverters = 3;     // codes
constexpr uint32_t kThreads = 12 * 32;  // 168 registers each at launch
// What the softmax warps, whose rows of 128 scores want more than that, take over from the
// other four: 8 x 32 x (208 - 168) = 4 x 32 x (168 - 88), codes 8 x 32 x (200 - 168) = 4 x
// 32 x (168 - 104), as the converters keep a batch of codes in registers. With 168 for all, 100
// to 290 bytes of spills: 8 x 1370 x 1370, 16 heads of 64, 143 us for 138; 700 queries over
// caches of up to 6000 tokens, 32 heads of 128, 149 us for 143.
template <bool kS8>
constexpr uint32_t kSoftmaxRegisters = kS8 ? 200 : 208;
template <bool kS8>
constexpr uint32_t kOtherRegisters = kS8 ? 104 : 88;
static_assert(2 * kSoftmaxRegisters<false> + kOtherRegisters<false> <= 3 * 168 &&
                  2 * kSoftmaxRegisters<true> + kOtherRegisters<true> <= 3 * 168,
              "more registers than the block is launched with");
// Warps that issue products: one for each tile, so that what one does between its
// products is hidden by the other's. Codes need the second warp for conversion.
template <int D, bool kS8>
constexpr uint32_t kIssuers = kS8 ? 1 : 2;
// At D = 128, where S waits for P, the two take turns: products that interleave bring the
// tiles into step, so that both softmaxes and then both products wait (128 x 5477 keys:
// 97 us, without turns 130 us). At D = 64, where S runs ahead, turns gain nothing.
template <int D>
constexpr bool kTurns = D == 128;

constexpr float kLowest = -3.402823466e38f;
template <int D, bool kS8>
struct Layout {
    static constexpr uint32_t kOperand = D / 64 * kAtom;   // bytes of 128 rows
    static constexpr uint32_t kQBufs = D == 64 && !kS8 ? 2 : 1;  // Q of this unit and the next
    static constexpr uint32_t kStages = kS8 ? (D == 64 ? 5 : 3) : (D == 64 ? 8 : 5);  // K or V tiles of 16 bits
    static constexpr uint32_t kRaw = kS8 ? 4 : 0;          // tiles of codes in flight
    static constexpr uint32_t kRawBytes = D * kKeys;
    static constexpr uint32_t kBars = 512;                 // bytes of barriers
    static constexpr uint32_t kSmem =
        (2 * kQBufs + kStages) * kOperand + kRaw * kRawBytes + kBars;
    // Tensor memory columns: S_0, S_1, O_0, O_1, and at D = 64 P_0, P_1; at D = 128,
    // where S and O fill it, P_t takes the first half of S_t.
    static constexpr bool kAlias = D == 128;
    static constexpr uint32_t kO = 256;
    static constexpr uint32_t kP = kAlias ? 0 : 384, kPStride = kAlias ? 128 : 64;
};
static_assert(Layout<128, false>::kSmem <= 232448 && Layout<64, false>::kSmem <= 232448 &&
                  Layout<128, true>::kSmem <= 232448 && Layout<64, true>::kSmem <= 232448,
              "shared memory above the per-block limit");

struct TilesParams {
    uint32_t takes_over;  // more units than SMs
    uint32_t q_box;  // Q by TMA: tokens of a 128-row box (0: by a warp)
    uint32_t slots, full_units, full_tiles;  // full_*: dense batches
};

// The products, from the low words of their descriptors (address and one stride);
// the high word is the same for all.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);  // 8-row stride, version 1, 128-byte swizzle
constexpr uint32_t kDescK = 1u << 16;             // K-major: no leading stride
constexpr uint32_t kDescV = (kAtom >> 4) << 16;   // MN-major: 64-dim groups one atom apart

template <bool kAccumulate>
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint32_t desc_a, uint32_t desc_b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(desc_a), "r"(desc_b), "r"(idesc), "n"(kAccumulate ? 1 : 0), "n"(kDescHigh)
        : "memory");
}

__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t desc_b, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "mov.b64 b, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "r"(desc_b), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
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

// 32 bytes of a row that starts on a 16-byte boundary: in one piece where they lie so. A lane
// has a row of its own, and what its stores cost is their number (131 us for 129).
__device__ __forceinline__ void store32(void* to, const uint32_t (&x)[8]) {
    if ((reinterpret_cast<uintptr_t>(to) & 31u) == 0) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]),
                     "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(to)[0] = make_uint4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<uint4*>(to)[1] = make_uint4(x[4], x[5], x[6], x[7]);
    }
}

// The largest of three; NaN if one is.
__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A block's next unit, by taking over the place of a block that has not started:
// the hardware writes its index, or that there is none, and completes 16 bytes on the barrier.
__device__ __forceinline__ void request_unit(uint4* response, uint64_t* bar) {
    asm volatile(
        "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
            smem_addr(response)),
        "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ bool read_unit(const uint4* response, uint32_t& unit) {
    uint32_t taken, x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t.reg .b32 y, z, w;\n\t"
        "ld.shared.b128 r, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, r;\n\t}"
        : "=r"(taken), "=r"(x)
        : "r"(smem_addr(response))
        : "memory");
    unit = x;
    return taken != 0;
}

// Byte of (row, 8-dim chunk) in a swizzled operand.
__device__ __forceinline__ uint32_t chunk_at(uint32_t row, uint32_t chunk) {
    return (chunk >> 3) * kAtom + row * 128u + (((chunk & 7u) ^ (row & 7u)) << 4);
}

// One unit of work: 256 rows of a sequence and key head, and a split of its keys.
struct Unit {
    RowTile where;
    uint32_t kv_head, split, len, row0, tiles, first, blocks;
    bool any;
};

// Units are numbered row tile first, then key head, then split, so that blocks that run
// together share K and V in L2. Dense batches: the full tiles of all sequences, then
// their last ones, which are shorter.
__device__ __forceinline__ Unit unit_at(const RowsParams& p, const TilesParams& n, uint32_t u) {
    Unit w;
    w.where = RowTile{};
    if (p.query_begin) {
        const uint32_t slot = u % n.slots, x = u / n.slots;
        w.kv_head = x % p.kv_heads;
        w.split = x / p.kv_heads;
        w.any = find_row_tile(w.where, p, slot, 2 * kTileRows);
    } else {
        uint32_t x;
        if (u < n.full_units) {
            x = u / n.full_tiles;
            w.where.tile = u - x * n.full_tiles;
        } else {
            x = u - n.full_units;
            w.where.tile = n.full_tiles;
        }
        w.kv_head = x % p.kv_heads;
        x /= p.kv_heads;
        w.where.seq = x % p.sequences;
        w.split = x / p.sequences;
        w.where.q_count = p.queries;
        w.where.rows = p.queries * p.group;
        w.any = true;
    }
    w.blocks = 0;
    if (!w.any) return w;
    w.len = keys_of(p, w.where.seq);
    w.row0 = w.where.tile * 2 * kTileRows;
    w.tiles = w.where.rows - w.row0 > kTileRows ? 2u : 1u;
    // the key blocks of this split, up to the last row's reach
    const uint32_t reach = reach_of(p, w.where, w.len, min(w.where.rows, w.row0 + 2 * kTileRows) - 1);
    const uint32_t all = (w.len + kKeys - 1) / kKeys, per_split = (all + p.splits - 1) / p.splits;
    w.first = w.split * per_split;
    const uint32_t last = min(min(all, w.first + per_split), (reach + kKeys - 1) / kKeys);
    w.blocks = last > w.first ? last - w.first : 0;
    return w;
}

template <int D, bool kS8, bool kBF16>
__global__ void __launch_bounds__(kThreads, 1)
    attention_tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, const RowsParams p, const TilesParams n) {
    using L = Layout<D, kS8>;
    constexpr uint32_t kStages = L::kStages;
    constexpr uint32_t kQBufs = L::kQBufs;
    extern __shared__ uint8_t smem[];
    uint8_t* sQ = smem;                        // [tile]
    uint8_t* sKV = smem + 2 * kQBufs * L::kOperand;  // [stage]
    uint8_t* sRaw = sKV + kStages * L::kOperand;     // [raw slot] codes, rows of head_dim bytes
    uint8_t* control = sRaw + L::kRaw * L::kRawBytes;
    uint4* response = reinterpret_cast<uint4*>(control);  // [2]
    uint64_t* full = reinterpret_cast<uint64_t*>(response + 2);  // [stage]
    uint64_t* empty = full + kStages;    // [stage]
    uint64_t* s_full = empty + kStages;  // [tile]
    uint64_t* s_free = s_full + 2;       // [tile]: S is in registers (P beside S)
    uint64_t* p_full = s_free + 2;       // [tile]
    uint64_t* pv_done = p_full + 2;      // [tile]
    uint64_t* o_full = pv_done + 2;      // [tile]
    uint64_t* q_full = o_full + 2;       // [buffer]; codes: [tile]
    uint64_t* q_empty = q_full + 2;      // [buffer]
    uint64_t* unit_full = q_empty + 2;   // [response]
    uint64_t* unit_empty = unit_full + 2;  // [response]
    uint64_t* turn = unit_empty + 2;     // [tile]
    uint64_t* drain = turn + 2;
    uint64_t* raw_full = drain + 2;      // codes: [raw slot]
    uint64_t* raw_empty = raw_full + 4;  // codes: [raw slot]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_empty + 4);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert(32 + 8 * (2 * kStages + 30) + 32 <= L::kBars, "barriers overflow their part");
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if ((smem_addr(smem) & 1023u) != 0) {  // the 128-byte swizzle needs 1 KB aligned tiles
        if (threadIdx.x == 0) atomicExch(p.err, 2);
        return;
    }
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kStages; ++i) {
            mbar_init(&full[i], kS8 ? kConverters : 1);
            mbar_init(&empty[i], kIssuers<D, kS8>);
        }
        for (uint32_t t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&s_free[t], 4);
            mbar_init(&p_full[t], 4);
            mbar_init(&pv_done[t], 1);
            mbar_init(&o_full[t], 1);
            mbar_init(&turn[t], 1);
            mbar_init(&q_full[t], kS8 ? 4 : 1);
            mbar_init(&q_empty[t], kIssuers<D, kS8>);
            mbar_init(&unit_full[t], 1);
            mbar_init(&unit_empty[t], kSoftmaxWarps + kIssuers<D, kS8> + (kS8 ? kConverters : 2));  // warps at work
        }
        for (uint32_t i = 0; kS8 && i < 4; ++i) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], kConverters);
        }
        mbar_init(&drain[0], 1);
        mbar_init(&drain[1], 1);
        *abort_flag = 0;
        fence_barrier_init();
        if (!kS8) {
            if (n.q_box) tma_prefetch_desc(&tm_q);
            tma_prefetch_desc(&tm_k);
            tma_prefetch_desc(&tm_v);
        }
    }
    if (warp == kSoftmaxWarps) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool mma_issued = false;
    // a warp's lanes leave a wait together: the collective accesses below never diverge
    auto warp_wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity & 1u, abort_flag, p.err));
    };

    // The unit after the `iter`-th one of this block; false: there is none (or a timeout).
    auto next_unit = [&](uint32_t iter, uint32_t& u) -> bool {
        if (!n.takes_over) return false;
        const uint32_t slot = iter & 1u;
        if (!warp_wait(&unit_full[slot], iter >> 1)) return false;
        const bool more = read_unit(&response[slot], u);
        __syncwarp();
        if (lane == 0) mbar_arrive(&unit_empty[slot]);
        return more;
    };
    // Asks for it (one thread), once every warp has read the response before the last. Not
    // at a unit's beginning: a block that has not started may be about to, on an idle SM.
    auto ask = [&](uint32_t iter) -> bool {
        if (!n.takes_over) return true;
        const uint32_t slot = iter & 1u;
        if (!mbar_wait(&unit_empty[slot], ((iter >> 1) & 1u) ^ 1u, abort_flag, p.err)) return false;
        fence_async_smem();
        mbar_arrive_expect_tx(&unit_full[slot], 16);
        request_unit(&response[slot], &unit_full[slot]);
        return true;
    };

    if (warp < kSoftmaxWarps) {
        // ------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters<kS8>));
        const uint32_t t = warp >> 2, quarter = warp & 3u;
        const uint32_t r = quarter * 32u + lane;  // row of the tile
        const uint32_t lanes = (quarter * 32u) << 16;
        const uint32_t tS = tmem + t * 128u + lanes, tP = tmem + L::kP + t * L::kPStride + lanes;
        const uint32_t tO = tmem + L::kO + t * D + lanes;
        uint32_t done = 0;   // blocks of this tile so far
        uint32_t outs = 0;   // units of this tile so far
        bool ok = true;
        uint32_t u = blockIdx.x;
        Unit next = unit_at(p, n, u);
        bool more = true, looked = true;  // of the next unit, found while the last product runs
        for (uint32_t iter = 0;; ++iter) {
            if (!looked) {
                more = next_unit(iter - 1, u);
                if (more) next = unit_at(p, n, u);
            }
            if (!more) break;
            looked = false;
            const Unit w = next;
            if (!w.any) {
                if (!iter) break;
                continue;
            }
            const uint32_t row = w.row0 + t * kTileRows + r;  // row of the sequence
            const bool live = row < w.where.rows;
            if (!w.blocks) {  // no key in reach
                if (t < w.tiles && live) {
                    if (p.splits > 1) {
                        p.part_ml[part_at(p, w.where, w.kv_head, row, w.split)] = make_float2(kLowest, 0.0f);
                    } else {
                        const uint64_t at = row_at(p, w.where, w.kv_head, row, p.out_batch, p.out_stride);
                        const float zero[2] = {0.0f, 0.0f};
                        for (uint32_t i = 0; i < p.head_dim; i += 2) store_out(p, at + i, zero, 2);
                    }
                }
                if (!iter) break;
                continue;
            }
            if (t >= w.tiles) continue;
            // a negative scale is in the first product's sign; 16-bit rows multiply by 0 where the mask is, whose
            // -inf would not outlast it, and then by 1
            const float once = kS8 || p.scale_log2 != 0.0f ? 1.0f : 0.0f;
            float c = once != 0.0f ? fabsf(p.scale_log2) : 1.0f;
            if constexpr (kS8) {
                // this row of Q, brought into f16's range by a power of two. The last unit's
                // products are done: this warp has waited for its output.
                const uint16_t* q = static_cast<const uint16_t*>(p.q) +
                                    (live ? row_at(p, w.where, w.kv_head, row, p.q_batch, p.q_stride) : 0);
                uint4 x[D / 8];
#pragma unroll
                for (int i = 0; i < D / 8; ++i)
                    x[i] = live && 8 * i < p.head_dim ? *reinterpret_cast<const uint4*>(q + 8 * i) : make_uint4(0, 0, 0, 0);
                uint32_t* y = reinterpret_cast<uint32_t*>(x);
                float most = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 2; ++i) {
                    const float2 v = unpack2(y[i], p.q_bf16);
                    most = fmaxf(most, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
                int ex = most > 0.0f ? 141 - (int)(__float_as_uint(most) >> 23) : 0;  // an infinity: all finite ones stay so
                ex = max(-120, min(120, ex));
                const float up = __uint_as_float((uint32_t)(127 + ex) << 23);
                c *= __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
                for (int i = 0; i < D / 2; ++i) {
                    const float2 v = unpack2(y[i], p.q_bf16);
                    y[i] = pack2<false>(v.x * up, v.y * up);
                }
#pragma unroll
                for (int i = 0; i < D / 8; ++i) *reinterpret_cast<uint4*>(sQ + t * L::kOperand + chunk_at(r, i)) = x[i];
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[t]);
            }
            // where the row's result goes, found now: the unit's numbers need no registers later
            const uint64_t at = !live ? 0
                                : p.splits > 1 ? part_at(p, w.where, w.kv_head, row, w.split)
                                               : row_at(p, w.where, w.kv_head, row, p.out_batch, p.out_stride);
            const uint32_t reach = reach_of(p, w.where, w.len, row);
            // the first key that a row of the warp does not see; all keys go through the mask where `once` is 0
            const uint32_t low = once == 0.0f ? 0u : __reduce_min_sync(0xffffffffu, live ? reach : 0xFFFFFFFFu);
            // codes: lane i has the K scale (i < 8), lane 8 + i the V scale, of the block's keys
            // 16i .. 16i + 15; fetched a block ahead. -1: no such page
            auto scale_of = [&](uint32_t j) -> float {
                const uint32_t key = (w.first + j) * kKeys + 16u * (lane & 7u);
                if (lane >= 16 || key >= w.len) return 0.0f;
                const int32_t page = p.page_table[(uint64_t)w.where.seq * p.table_stride + (key >> p.page_shift)];
                if (page < 0 || (uint32_t)page >= p.pages) return lane < 8 ? -1.0f : 0.0f;
                const uint64_t unit = (uint64_t)page * p.kv_heads + w.kv_head;
                return (lane < 8 ? p.k_scales : p.v_scales)[unit];
            };
            float scale_next = 0.0f, scale_now = 0.0f, v_shift = 0.0f, v_weight = 0.0f, v_back = 0.0f;
            if constexpr (kS8) scale_next = scale_of(0);
            float m = kLowest, l = 0.0f;
            // f16: P is kept times 2^7, which leaves f16 down to 2^-31 of the row's largest
            constexpr float kShift = kBF16 || kS8 ? 0.0f : 7.0f;
            for (uint32_t j = 0; j < w.blocks; ++j, ++done) {
                if (!warp_wait(&s_full[t], done)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                uint32_t sr[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(tS + 32u * i, sr[i]);
                tmem_ld_wait();
                if constexpr (!L::kAlias) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[t]);
                }
                float s[128];
#pragma unroll
                for (int i = 0; i < 128; ++i) s[i] = __uint_as_float(sr[i >> 5][i & 31]);
                const uint32_t key0 = (w.first + j) * kKeys;
                if constexpr (kS8) {
                    scale_now = scale_next;
                    if (j + 1 < w.blocks) scale_next = scale_of(j + 1);
                    split_scale(fmaxf(scale_now, 0.0f), v_shift, v_weight, v_back);  // lanes 8 to 15
                    v_weight *= 128.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float f = __shfl_sync(0xffffffffu, scale_now, i) * c;
                        const float shift = __shfl_sync(0xffffffffu, v_shift, 8 + i);
#pragma unroll
                        for (int e = 16 * i; e < 16 * i + 16; e += 2)
                            f2_fma(s[e], s[e + 1], s[e], s[e + 1], f, f, shift, shift);
                    }
                    if (__any_sync(0xffffffffu, scale_now < 0.0f)) {  // keys of no page of the cache
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (__shfl_sync(0xffffffffu, scale_now, i) < 0.0f) {
#pragma unroll
                                for (int e = 0; e < 16; ++e) s[16 * i + e] = -INFINITY;
                            }
                    }
                }
                if (key0 + kKeys > low) {
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        s[i] = key0 + i >= reach ? -INFINITY : kS8 ? s[i] : s[i] * once;
                }
                // four chains: a tree's partial maxima beside 128 scores would not fit the registers
                float a[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < 124; i += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] = fmax3(a[e], s[i + 2 * e], s[i + 2 * e + 1]);
                a[0] = fmax3(a[0], s[124], s[125]), a[1] = fmax3(a[1], s[126], s[127]);
                float top = fmax3(fmax3(a[0], a[1], a[2]), a[3], a[3]);
                if constexpr (!kS8) top = top == -INFINITY ? top : top * c;
                // P's columns, and O, are free once the product of the block before is done: waited for
                // where they are written (before the maximum's vote: 138 us for 134)
                auto last_product = [&]() -> bool {
                    const bool done_now = warp_wait(&pv_done[t], done - 1);
                    tc_fence_after();
                    return done_now;
                };
                const bool raise = top > m + kRaise<kS8>;
                if (__any_sync(0xffffffffu, raise)) {
                    const float up = fmaxf(m, top);
                    const float down = ex2_approx(m - up);
                    if (j > 0) {  // with P in S's columns, P V was issued before this S
                        if (!L::kAlias) ok = last_product();
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
                const float off = kShift - m;
                float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t x2[32];
                    float part[4];  // codes: sum over the 16 keys of a V scale
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float x = s[64 * h + 2 * i], y = s[64 * h + 2 * i + 1];
                        if constexpr (kS8) f2_add(x, y, x, y, off, off);
                        else f2_fma(x, y, x, y, c, c, off, off);
                        x = ex2_approx(x), y = ex2_approx(y);
                        if constexpr (kS8) {
                            constexpr int kPairs = 8;
                            const int e = 2 * (i & 1);
                            if (i % kPairs < 2) part[e] = x, part[e + 1] = y;
                            else f2_add(part[e], part[e + 1], part[e], part[e + 1], x, y);
                            const float weight = __shfl_sync(0xffffffffu, v_weight, 8 + 4 * h + i / kPairs);
                            f2_mul(x, y, x, y, weight, weight);
                            if (i % kPairs == kPairs - 1) {
                                const float back = __shfl_sync(0xffffffffu, v_back, 8 + 4 * h + i / kPairs);
                                f2_fma(ls[0], ls[1], part[0], part[1], back, back, ls[0], ls[1]);
                                f2_fma(ls[2], ls[3], part[2], part[3], back, back, ls[2], ls[3]);
                            }
                        } else {
                            f2_add(ls[(2 * i) & 3], ls[(2 * i + 1) & 3], ls[(2 * i) & 3], ls[(2 * i + 1) & 3], x, y);
                        }
                        x2[i] = pack2<kBF16>(x, y);
                    }
                    if (!L::kAlias && h == 0 && j > 0) ok = last_product() && ok;
                    tmem_st_32x32b_x32(tP + 32u * h, x2);
                }
                if (!ok) break;
                l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            if (!ok) break;
            more = next_unit(iter, u);
            if (more) next = unit_at(p, n, u);
            looked = true;
            if (!warp_wait(&o_full[t], outs++)) break;
            tc_fence_after();
            constexpr float unit_v = kS8 ? 1.0f / 128.0f : 1.0f;
            const float back = kShift != 0.0f ? 1.0f / 128.0f : 1.0f;
            const float f = l != 0.0f ? (p.splits == 1 ? unit_v / l : unit_v * back) : 0.0f;
            if (live && p.splits > 1) p.part_ml[at] = make_float2(m, l * back);
#pragma unroll 1
            for (uint32_t k = 0; k < D / 32; ++k) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(tO + 32u * k, o);
                tmem_ld_wait();
                if (!live) continue;
#pragma unroll
                for (int i = 0; i < 32; i += 16) {
                    const uint32_t dim = 32 * k + i;
                    if (dim >= p.head_dim) continue;
                    const bool whole = dim + 16 <= p.head_dim;  // else 8 dims
                    float x[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = l != 0.0f ? __uint_as_float(o[i + e]) * f : 0.0f;
                    uint32_t y[8];
                    if (p.splits > 1 || p.out_kind == 0) {
                        float* to = (p.splits > 1 ? p.part_o + at * p.head_dim : static_cast<float*>(p.out) + at) + dim;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (h && !whole) continue;
#pragma unroll
                            for (int e = 0; e < 8; ++e) y[e] = __float_as_uint(x[8 * h + e]);
                            store32(to + 8 * h, y);
                        }
                    } else {
                        uint16_t* to = static_cast<uint16_t*>(p.out) + at + dim;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            y[e] = p.out_kind == 1 ? pack2<true>(x[2 * e], x[2 * e + 1])
                                                   : pack2<false>(x[2 * e], x[2 * e + 1]);
                        if (whole) store32(to, y);
                        else *reinterpret_cast<uint4*>(to) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                }
            }
            tc_fence_before();  // O is read: the next unit's first product, after its P, may overwrite it
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters<kS8>));
        if (warp < kSoftmaxWarps + kIssuers<D, kS8>) {
            // ----------------------------------------------------------- products
            // One thread issues, with everything but the waits unrolled: between its products the
            // tensor cores may wait, as their queue holds a few (rolled up, 5 to 15% slower).
            constexpr uint32_t ab = kBF16 ? 1u : 0u;
            const uint32_t idesc_s = make_idesc(1u, ab, 128u, 128u) | (p.scale_log2 < 0.0f ? 1u << 13 : 0u);  // or -Q
            constexpr uint32_t idesc_o = make_idesc(1u, ab, 128u, D) | (1u << 16);  // V is MN-major
            constexpr uint32_t kStageDesc = L::kOperand >> 4;
            const uint32_t kv_base = smem_addr(sKV) >> 4, q_all = (smem_addr(sQ) >> 4) | kDescK;
            const uint32_t role = warp - kSoftmaxWarps;
            uint32_t units = 0, stage = 0, phase = 0;  // stage and phase of the unit's next tile in the ring
            uint32_t done0 = 0, done1 = 0;             // blocks of each tile before this unit
            uint32_t turns = 0, pairs = 0;             // blocks of units with two tiles; such units
            auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
                return mbar_wait(bar, parity & 1u, abort_flag, p.err);
            };
            auto next_stage = [&](uint32_t by) {
                stage += by;
                if (stage >= kStages) stage -= kStages, phase ^= 1u;
            };
            auto issue_s = [&](uint32_t t, uint32_t q, uint32_t st) {
                q += t * kStageDesc;
                const uint32_t k = kv_base + st * kStageDesc + kDescK, d = tmem + 128u * t;
                umma_ss<false>(d, q, k, idesc_s);
#pragma unroll
                for (uint32_t kk = 1; kk < D / 16; ++kk) {
                    const uint32_t off = ((kk / 4) * kAtom + 32u * (kk % 4)) >> 4;
                    umma_ss<true>(d, q + off, k + off, idesc_s);
                }
                umma_commit(&s_full[t]);
            };
            auto issue_o = [&](uint32_t t, uint32_t st, uint32_t steps, uint32_t later) {
                const uint32_t o = tmem + L::kO + t * D, pt = tmem + L::kP + t * L::kPStride;
                const uint32_t v = kv_base + st * kStageDesc + kDescV;
                if (steps == 8) {
                    umma_ts(o, pt, v, idesc_o, later);
#pragma unroll
                    for (uint32_t kk = 1; kk < 8; ++kk) umma_ts(o, pt + 8u * kk, v + 128u * kk, idesc_o, 1u);
                } else {
                    for (uint32_t kk = 0; kk < steps; ++kk) umma_ts(o, pt + 8u * kk, v + 128u * kk, idesc_o, later | kk);
                }
            };
            // rows of V behind the last key, up to the product's end
            auto clear_tail = [&](uint32_t st, uint32_t valid) {
                uint8_t* v = sKV + st * L::kOperand;
#pragma unroll 1
                for (uint32_t i = 0; i < (16u - (valid & 15u)) * (D / 8); ++i)
                    *reinterpret_cast<uint4*>(v + chunk_at(valid + i / (D / 8), i % (D / 8))) = make_uint4(0, 0, 0, 0);
                fence_async_smem();
            };
            uint32_t u = blockIdx.x;
            for (uint32_t iter = 0;; ++iter) {
                if (iter && !next_unit(iter - 1, u)) break;
                const Unit w = unit_at(p, n, u);
                if (!w.blocks) {
                    if (!iter) break;
                    continue;
                }
                const uint32_t qb = units % kQBufs, q = q_all + qb * 2 * kStageDesc;
                const uint32_t tiles = w.tiles, blocks = w.blocks;
                const uint32_t last_keys = min(kKeys, w.len - (w.first + blocks - 1) * kKeys);  // of the last block
                bool ok = true;
                if (lane == 0) {
                    mma_issued = true;
                    const uint32_t t0 = kIssuers<D, kS8> == 2 ? role : 0;
                    const uint32_t t1 = kIssuers<D, kS8> == 2 ? min(t0 + 1, tiles) : tiles;
                    const bool take_turns = kTurns<D> && kIssuers<D, kS8> == 2 && tiles == 2;
                    ok = (kS8 || wait(&q_full[qb], units / kQBufs)) && wait(&full[stage], phase);
#pragma unroll 1
                    for (uint32_t t = t0; t < t1 && ok; ++t) {
                        if (kS8) ok = wait(&q_full[t], t ? pairs : units);
                        const uint32_t before = t ? done1 : done0;
                        if (!L::kAlias && before) ok = ok && wait(&s_free[t], before - 1);
                        tc_fence_after();
                        if (ok) issue_s(t, q, stage);
                    }
                    if (t0 < t1) {
                        umma_commit(&empty[stage]);
                        if (blocks == 1) umma_commit(&q_empty[qb]);
                    } else if (ok) {  // no rows of this tile: its stages are released as they are filled
                        mbar_arrive(&empty[stage]);
                        mbar_arrive(&q_empty[qb]);
                    }
                    next_stage(1);
#pragma unroll 1
                    for (uint32_t j = 0; ok && j < blocks; ++j) {
                        const bool more = j + 1 < blocks;
                        const uint32_t sv = stage;
                        ok = wait(&full[sv], phase);
                        next_stage(1);
                        const uint32_t sk = stage;
                        if (more) {
                            ok = ok && wait(&full[sk], phase);
                            next_stage(1);
                        }
                        if (t0 >= t1) {
                            if (!ok) break;
                            mbar_arrive(&empty[sv]);
                            if (more) mbar_arrive(&empty[sk]);
                            continue;
                        }
                        const uint32_t valid = more ? kKeys : last_keys;
                        if (ok && !kS8 && (valid & 15u)) clear_tail(sv, valid);
                        // S of the next block: beside this block's softmax where P has its own columns
                        if (!L::kAlias && more) {
#pragma unroll 1
                            for (uint32_t t = t0; t < t1 && ok; ++t) {
                                ok = wait(&s_free[t], (t ? done1 : done0) + j);
                                tc_fence_after();
                                if (ok) issue_s(t, q, sk);
                            }
                            umma_commit(&empty[sk]);
                            if (j + 2 == blocks) umma_commit(&q_empty[qb]);
                        }
#pragma unroll 1
                        for (uint32_t t = t0; t < t1 && ok; ++t) {
                            ok = wait(&p_full[t], (t ? done1 : done0) + j);
                            // the tiles' products one after the other, not interleaved: tile 0 of
                            // block j, tile 1 of block j, tile 0 of block j + 1
                            if (take_turns && ok && (t || turns + j)) ok = wait(&turn[t], t ? turns + j : turns + j - 1);
                            tc_fence_after();
                            if (!ok) break;
                            issue_o(t, sv, (valid + 15u) / 16u, j);
                            if (L::kAlias && more) issue_s(t, q, sk);
                            if (take_turns) mbar_arrive(&turn[t ^ 1u]);
                            if (!L::kAlias) umma_commit(&pv_done[t]);
                            if (!more) umma_commit(&o_full[t]);
                        }
                        umma_commit(&empty[sv]);
                        if (L::kAlias && more) {
                            umma_commit(&empty[sk]);
                            if (j + 2 == blocks) umma_commit(&q_empty[qb]);
                        }
                    }
                }
                done0 += blocks;
                if (tiles == 2) done1 += blocks, turns += blocks, ++pairs;
                ++units;
                __syncwarp();
                if (!__shfl_sync(0xffffffffu, ok, 0)) break;
            }
        } else if constexpr (!kS8) {
            uint32_t ring = 0, units = 0;
            if (warp == 10) {
                // -------------------------------------------------- TMA, and the next unit
                uint32_t u = blockIdx.x;
                for (uint32_t iter = 0;; ++iter) {
                    if (iter && !next_unit(iter - 1, u)) break;
                    const Unit w = unit_at(p, n, u);
                    bool ok = true;
                    if (lane == 0) {
                        const int k_batch = p.k_batch ? (int)w.where.seq : 0, v_batch = p.v_batch ? (int)w.where.seq : 0;
                        if (!w.blocks) ok = iter && ask(iter);  // a block whose first unit is empty leaves
                        for (uint32_t i = 0; i < 2 * w.blocks; ++i) {
                            const uint32_t at = ring + i, st = at % kStages;
                            if (i == min(kStages + 1, 2 * w.blocks - 1)) ok = ask(iter);
                            if (!ok || *abort_flag || !mbar_wait(&empty[st], ((at / kStages) & 1u) ^ 1u, abort_flag, p.err)) {
                                ok = false;
                                break;
                            }
                            mbar_arrive_expect_tx(&full[st], L::kOperand);
                            const int key0 = (int)((w.first + i / 2) * kKeys);
#pragma unroll
                            for (int h = 0; h < D / 64; ++h)
                                tma_load_4d(sKV + st * L::kOperand + h * kAtom, i & 1 ? &tm_v : &tm_k, &full[st], 64 * h,
                                            (int)w.kv_head, key0, i & 1 ? v_batch : k_batch);
                        }
                    }
                    if (!__shfl_sync(0xffffffffu, ok, 0)) break;
                    ring += 2 * w.blocks;
                }
            } else if (warp == 11) {
                // -------------------------------------------------------------- Q
                uint32_t u = blockIdx.x;
                for (uint32_t iter = 0;; ++iter) {
                    if (iter && !next_unit(iter - 1, u)) break;
                    const Unit w = unit_at(p, n, u);
                    if (!w.blocks) {
                        if (!iter) break;
                        continue;
                    }
                    const uint32_t qb = units % kQBufs;
                    if (!warp_wait(&q_empty[qb], (units / kQBufs) ^ 1u)) break;
                    ++units;
                    uint8_t* to = sQ + qb * 2 * L::kOperand;
                    if (n.q_box) {
                        // 128 rows are q_box tokens of the group's heads
                        if (lane == 0) {
                            mbar_arrive_expect_tx(&q_full[qb], w.tiles * L::kOperand);
                            const int batch = p.q_batch ? (int)w.where.seq : 0;
                            for (uint32_t t = 0; t < w.tiles; ++t)
#pragma unroll
                                for (int h = 0; h < D / 64; ++h)
                                    tma_load_4d(to + t * L::kOperand + h * kAtom, &tm_q, &q_full[qb], 64 * h,
                                                (int)(w.kv_head * p.group), (int)((w.where.tile * 2 + t) * n.q_box), batch);
                        }
                        __syncwarp();
                        continue;
                    }
                    const uint32_t rows = w.tiles * kTileRows;
#pragma unroll 1
                    for (uint32_t i = lane; i < rows * (D / 8); i += 32) {
                        const uint32_t r = i / (D / 8), chunk = i % (D / 8), row = w.row0 + r;
                        const bool read = row < w.where.rows && 8 * chunk < p.head_dim;
                        const uint16_t* from = static_cast<const uint16_t*>(p.q) +
                                               (read ? row_at(p, w.where, w.kv_head, row, p.q_batch, p.q_stride) + 8 * chunk : 0);
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                         smem_addr(to + (r / kTileRows) * L::kOperand + chunk_at(r % kTileRows, chunk))),
                                     "l"(from), "r"(read ? 16u : 0u)
                                     : "memory");
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_full[qb]);
                }
            }
        } else {
            // -------------------------------------------------------------- codes
            // kRaw tiles of codes are under way from the pages (a page's tokens of a head are one
            // run of bytes, copied in one piece; the three warps start the copies in turn); the
            // warps turn each into a 16-bit tile, 16 dims of a key at a time.
            constexpr uint32_t kParts = D / 16, kStep = 32 * kConverters;
            const uint32_t i0 = threadIdx.x - 9 * 32;
            const uint32_t in_page = (1u << p.page_shift) - 1;
            uint32_t ring = 0;
            bool ok = true;
            uint32_t u = blockIdx.x;
            for (uint32_t iter = 0; ok; ++iter) {
                if (iter && !next_unit(iter - 1, u)) break;
                const Unit w = unit_at(p, n, u);
                if (!w.blocks) {
                    if (!iter) break;  // a block whose first unit is empty leaves
                    if (i0 == 0) ok = ask(iter);
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    continue;
                }
                // lanes 0 to 7 have the page of their piece of a block
                const uint32_t piece = min(1u << p.page_shift, kKeys);
                auto page_of = [&](uint32_t j) -> int32_t {
                    const uint32_t in_block = lane * piece, key = (w.first + j) * kKeys + in_block;
                    if (in_block >= kKeys || key >= w.len) return -1;
                    const int32_t page = p.page_table[(uint64_t)w.where.seq * p.table_stride + (key >> p.page_shift)];
                    if (page < 0 || (uint32_t)page >= p.pages) {
                        atomicExch(p.err, 3);
                        return -1;
                    }
                    return page;
                };
                const uint32_t count = 2 * w.blocks, turn_of = i0 / 32;
                int32_t page_next = turn_of < count ? page_of(turn_of / 2) : -1;  // for the warp's next tile
                // Starts the copies of tile i (K_j: 2j, V_j: 2j + 1). Keys of no page, and past the
                // end, keep what the slot holds: any byte is a finite code, and they weigh nothing.
                auto fetch = [&](uint32_t i) -> bool {
                    const uint32_t at = ring + i, slot = at % L::kRaw;
                    if (!warp_wait(&raw_empty[slot], (at / L::kRaw) ^ 1u)) return false;
                    const int32_t page_now = page_next;
                    if (i + kConverters < count) page_next = page_of((i + kConverters) / 2);
                    const uint32_t bytes = piece * p.head_dim;
                    const uint32_t live = __popc(__ballot_sync(0xffffffffu, page_now >= 0));
                    if (lane == 0) mbar_arrive_expect_tx(&raw_full[slot], live * bytes);
                    __syncwarp();
                    if (page_now >= 0) {
                        const uint32_t key = (w.first + i / 2) * kKeys + lane * piece;
                        const int8_t* from =
                            static_cast<const int8_t*>(i & 1 ? p.v : p.k) +
                            ((((uint64_t)page_now * p.kv_heads + w.kv_head) << p.page_shift) + (key & in_page)) * p.head_dim;
                        asm volatile(
                            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                smem_addr(sRaw + slot * L::kRawBytes + lane * bytes)),
                            "l"(from), "r"(bytes), "r"(smem_addr(&raw_full[slot]))
                            : "memory");
                    }
                    __syncwarp();
                    return true;
                };
                for (uint32_t i = turn_of; ok && i < min(count, L::kRaw); i += kConverters) ok = fetch(i);
                if (!ok) break;
                for (uint32_t i = 0; ok && i < count; ++i) {
                    const uint32_t at = ring + i, st = at % kStages, slot = at % L::kRaw;
                    ok = warp_wait(&raw_full[slot], at / L::kRaw) && warp_wait(&empty[st], (at / kStages) ^ 1u);
                    if (!ok) break;
                    uint8_t* to = sKV + st * L::kOperand;
                    const uint8_t* from = sRaw + slot * L::kRawBytes;
                    // a batch of loads ahead of its conversions and stores, which the compiler keeps in the
                    // order written (one by one: 143 us for 134)
                    constexpr uint32_t kPieces = (kKeys * kParts + kStep - 1) / kStep, kBatch = 4;
#pragma unroll
                    for (uint32_t k0 = 0; k0 < kPieces; k0 += kBatch) {
                        uint4 x[kBatch];
                        uint32_t key[kBatch], part[kBatch];
#pragma unroll
                        for (uint32_t k = 0; k < kBatch; ++k) {
                            // eight lanes: four dims' parts of two rows, at D = 128 the first half of one and
                            // the second of the other, which spreads loads and stores over the banks
                            const uint32_t at16 = i0 + kStep * (k0 + k);
                            key[k] = D == 64 ? at16 / 4 : at16 / 16 * 2 + (at16 / 4 & 1);
                            part[k] = D == 64 ? at16 % 4 : at16 % 4 + 4 * ((at16 / 4 ^ at16 / 8) & 1);
                            x[k] = make_uint4(0, 0, 0, 0);
                            if (key[k] < kKeys && 16 * part[k] < p.head_dim)
                                x[k] = *reinterpret_cast<const uint4*>(from + key[k] * p.head_dim + 16 * part[k]);
                        }
#pragma unroll
                        for (uint32_t k = 0; k < kBatch; ++k) {
                            if (key[k] >= kKeys) continue;
                            const uint32_t w4[4] = {x[k].x ^ 0x80808080u, x[k].y ^ 0x80808080u, x[k].z ^ 0x80808080u,
                                                    x[k].w ^ 0x80808080u};
                            *reinterpret_cast<uint4*>(to + chunk_at(key[k], 2 * part[k])) =
                                make_uint4(codes_lo(w4[0]), codes_hi(w4[0]), codes_lo(w4[1]), codes_hi(w4[1]));
                            *reinterpret_cast<uint4*>(to + chunk_at(key[k], 2 * part[k] + 1)) =
                                make_uint4(codes_lo(w4[2]), codes_hi(w4[2]), codes_lo(w4[3]), codes_hi(w4[3]));
                        }
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&full[st]);
                        mbar_arrive(&raw_empty[slot]);
                    }
                    if (i == min(4u, count - 1)) {
                        if (i0 == 0) ok = ask(iter);
                        ok = __shfl_sync(0xffffffffu, ok, 0);
                        if (!ok) break;
                    }
                    __syncwarp();
                    if (i + L::kRaw < count && (i + L::kRaw) % kConverters == turn_of) ok = fetch(i + L::kRaw);
                }
                ring += count;
            }
        }
    }

    __syncthreads();
    if (*abort_flag) {
        if (warp >= kSoftmaxWarps && warp < kSoftmaxWarps + kIssuers<D, kS8> && lane == 0 && mma_issued) {
            uint64_t* d = &drain[warp - kSoftmaxWarps];
            umma_commit(d);
            const unsigned long long t0 = globaltimer();
            while (!mbar_try_wait(smem_addr(d), 0) && globaltimer() - t0 < 100000000ull) {
            }
        }
        if (threadIdx.x == 0) {  // copies in flight land before the block's memory is given back
            const unsigned long long t0 = globaltimer();
            while (globaltimer() - t0 < 2000000ull) {
            }
        }
        __syncthreads();
    }
    if (warp == kSoftmaxWarps) {
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

// q [batch][queries][q_heads][head_dim] as boxes of 64 dims x the heads of a group x
// as many tokens as make 128 rows.
bool encode_queries(CUtensorMap& tm, const RowsParams& p, uint32_t tokens, bool bf16) {
    const uint64_t row = (uint64_t)p.kv_heads * p.group * p.head_dim;
    const bool batches = p.q_batch && p.sequences > 1;
    const cuuint64_t dims[4] = {p.head_dim, (cuuint64_t)p.kv_heads * p.group, p.queries, batches ? p.sequences : 1u};
    const cuuint64_t strides[3] = {p.head_dim * 2ull, (p.queries > 1 ? p.q_stride : row) * 2,
                                   (batches ? p.q_batch : row) * 2};
    const cuuint32_t box[4] = {64, p.group, tokens, 1}, each[4] = {1, 1, 1, 1};
    return g_encode(&tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                    const_cast<void*>(p.q), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kS8, bool kBF16>
int start(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const RowsParams& p, const TilesParams& n,
          uint32_t blocks, cudaStream_t st) {
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
    kernel<<<blocks, kThreads, L::kSmem, st>>>(q, k, v, p, n);
    return check_launch("attention_tiles");
}

}  // namespace

int launch_attention_tiles(const RowsParams& p, uint32_t slots, bool s8, bool bf16, cudaStream_t st) {
    CUtensorMap q{}, k{}, v{};
    TilesParams n{};
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
        // any other group: rows that a warp copies
        if (kTileRows % p.group == 0 && encode_queries(q, p, kTileRows / p.group, bf16)) n.q_box = kTileRows / p.group;
    }
    const uint64_t heads = (uint64_t)p.kv_heads * p.splits, rows = (uint64_t)p.queries * p.group;
    n.slots = slots;
    n.full_tiles = (uint32_t)(rows / (2 * kTileRows));
    const uint64_t full_units = p.query_begin ? 0 : heads * p.sequences * n.full_tiles;
    const uint64_t units = p.query_begin ? heads * slots
                                         : full_units + (rows % (2 * kTileRows) ? heads * p.sequences : 0);
    if (units > 0x7FFFFFFFu) return set_error(DAV2CUDA_INVALID_ARGUMENT, "attention: too many row tiles");
    n.full_units = (uint32_t)full_units;
    int dev = 0;
    cudaGetDevice(&dev);
    n.takes_over = units > (uint64_t)sm_count(dev);
    const bool small = p.head_dim <= 64;
    const uint32_t blocks = (uint32_t)units;
    if (s8) return small ? start<64, true, false>(q, k, v, p, n, blocks, st) : start<128, true, false>(q, k, v, p, n, blocks, st);
    if (bf16) return small ? start<64, false, true>(q, k, v, p, n, blocks, st) : start<128, false, true>(q, k, v, p, n, blocks, st);
    return small ? start<64, false, false>(q, k, v, p, n, blocks, st) : start<128, false, false>(q, k, v, p, n, blocks, st);
}

}  // namespace dav2cuda

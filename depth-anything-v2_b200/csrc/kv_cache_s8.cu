// Appending keys and values to a paged cache of int8 codes: pages
// [page][head][token][dim], one f32 scale for each page and head (of K and of V).
//
//   scale = max(absmax / 127, 1e-8), code = rint(clamp(x / scale, -127, 127))
//
// the rule of the int8 activations, over all values of a page and head. A page
// that already holds tokens keeps its scale while that covers the new rows;
// where they need a larger one, its codes become rint(code * (old / new)), the
// ratio rounded to f32. Infinities take the codes +-127 and NaN the code 0, and
// neither enters a scale.
//
// Bound by memory: the rows are read once, into registers, and the codes written once
// (20011 tokens of 5 prompts, 8 heads of 128, f16: 34 us, 3.7 TB/s; what is missing to the
// memory's rate is each block's own chain from its offsets over its page to its rows). One
// block for each page that receives tokens, each head, and K or V; the blocks of sequence s
// are numbered from floor(begin[s] / page_tokens) + 2 s, which leaves room for its pages
// whatever their boundaries, so that the host needs no length: blocks without a page leave
// at once.
#include <type_traits>

#include "abi_check.h"
#include "kernels.cuh"

namespace dav2cuda {
namespace {

constexpr uint32_t kMost = 8;  // vectors of eight values that a thread keeps in registers

struct AppendParams {
    int8_t* codes[2];  // K, V
    float* scales[2];
    const void* rows[2];
    uint64_t stride[2];
    const int32_t* page_table;
    const int32_t* cached;
    const int32_t* begin;
    uint32_t sequences, tokens, heads, head_dim, pages, page_shift, table_stride;
    int* err;
};

// Eight consecutive values as they lie in memory.
template <typename T>
struct Vector {
    uint4 u[sizeof(T) / 2];

    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) u[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
        const T* t = reinterpret_cast<const T*>(u);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(t[i]);
    }
    // The largest magnitude's bits so far, 16-bit values two to a word: magnitudes order as
    // their bits do, infinities and NaN above all others.
    __device__ __forceinline__ uint32_t largest(uint32_t most) const {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
            const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 4) most = max(most, w[e] & 0x7FFFFFFFu);
                else most = __vmaxu2(most, w[e] & 0x7FFF7FFFu);
            }
        }
        return most;
    }
};

// A magnitude from its bits.
template <typename T>
__device__ __forceinline__ float from_bits(uint32_t bits) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
    else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)bits));
    else return __uint_as_float(bits << 16);
}

template <typename T, uint32_t kThreads>
__global__ void __launch_bounds__(kThreads) kv_cache_append_kernel(const AppendParams p) {
    // K and V of a token's heads lie side by side: neighbouring blocks read neighbouring bytes
    const uint32_t slot = blockIdx.x / (2 * p.heads), which = blockIdx.x / p.heads % 2, head = blockIdx.x % p.heads;
    const uint32_t page_tokens = 1u << p.page_shift;
    // the last sequence whose blocks begin at or before this one
    const uint32_t s = warp_last_at_most(p.sequences, slot, [&](uint32_t i) {
        return (uint64_t)((uint32_t)p.begin[i] >> p.page_shift) + 2 * i;
    });
    const int64_t begin = p.begin[s], end = p.begin[s + 1], cached = p.cached[s];
    const int64_t j = (int64_t)slot - ((begin >> p.page_shift) + 2 * (int64_t)s);
    if (j < 0) return;  // rows before the first sequence
    if (begin < 0 || end < begin || end > (int64_t)p.tokens || cached < 0) {
        if (threadIdx.x == 0 && head == 0) atomicExch(p.err, 3);
        return;
    }
    const int64_t page_at = (cached >> p.page_shift) + j;           // page of the sequence
    const int64_t first = max(cached, page_at << p.page_shift);     // its tokens that are new here
    const int64_t last = min(cached + end - begin, (page_at + 1) << p.page_shift);
    if (first >= last) return;
    const int32_t page = page_at < p.table_stride ? p.page_table[(uint64_t)s * p.table_stride + page_at] : -1;
    if (page < 0 || (uint32_t)page >= p.pages) {
        if (threadIdx.x == 0 && head == 0) atomicExch(p.err, 3);
        return;
    }
    const uint32_t held = (uint32_t)(first & (page_tokens - 1));
    const uint32_t count = (uint32_t)(last - first);
    const uint32_t per_row = p.head_dim / 8;
    const T* rows = static_cast<const T*>(p.rows[which]) + (uint64_t)(begin + first - cached) * p.stride[which] +
                    (uint64_t)head * p.head_dim;
    const uint64_t unit = (uint64_t)page * p.heads + head;
    int8_t* codes = p.codes[which] + ((unit << p.page_shift) * p.head_dim);

    // The rows of the page: in registers where a thread has at most kMost vectors of them,
    // all loads under way at once; else (a short block's long page) read again below.
    const uint32_t vectors = count * per_row;
    const uint32_t inverse_row = (65535 + per_row) / per_row;  // i / per_row of i < 65536 / 16
    const bool once = vectors <= kThreads * kMost;
    auto at = [&](uint32_t i) -> const T* {
        const uint32_t row = (i * inverse_row) >> 16;
        return rows + row * p.stride[which] + (i - row * per_row) * 8;
    };
    Vector<T> x[kMost];
    uint32_t bits = 0;
    for (uint32_t base = threadIdx.x; base < vectors; base += kThreads * kMost) {
#pragma unroll
        for (uint32_t k = 0; k < kMost; ++k) {
            const uint32_t i = base + k * kThreads;
            if (i < vectors) x[k].load(at(i));
            else x[k].clear();
        }
#pragma unroll
        for (uint32_t k = 0; k < kMost; ++k) bits = x[k].largest(bits);
    }
    if constexpr (sizeof(T) == 2) bits = max(bits & 0xFFFFu, bits >> 16);
    bits = __reduce_max_sync(0xffffffffu, bits);
    __shared__ uint32_t s_bits[kThreads / 32];
    if ((threadIdx.x & 31) == 0) s_bits[threadIdx.x / 32] = bits;
    const float old = held ? p.scales[which][unit] : 0.0f;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 32; ++w) bits = max(bits, s_bits[w]);
    float most = from_bits<T>(bits);
    const bool odd = !(most < INFINITY);  // an infinity or NaN: the largest finite magnitude, the long way
    if (odd) {
        most = 0.0f;
        for (uint32_t i = threadIdx.x; i < vectors; i += kThreads) {
            Vector<T> y;
            y.load(at(i));
            float f[8];
            y.floats(f);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[e]) < INFINITY ? fabsf(f[e]) : 0.0f);
        }
        most = warp_max(most);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s_bits[threadIdx.x / 32] = __float_as_uint(most);
        __syncthreads();
        for (uint32_t w = 0; w < kThreads / 32; ++w) most = fmaxf(most, __uint_as_float(s_bits[w]));
    }
    const float need = fmaxf(__fdiv_rn(most, 127.0f), 1e-8f);
    const bool grows = held == 0 || need > old;
    const float scale = grows ? need : old;
    if (grows && held) {
        const float ratio = __fdiv_rn(old, scale);
        for (uint32_t i = threadIdx.x; i < held * per_row; i += kThreads) {
            int2 c = reinterpret_cast<const int2*>(codes)[i];
            int8_t* b = reinterpret_cast<int8_t*>(&c);
#pragma unroll
            for (int e = 0; e < 8; ++e) b[e] = (int8_t)__float2int_rn(__fmul_rn((float)b[e], ratio));
            reinterpret_cast<int2*>(codes)[i] = c;
        }
    }
    const float inverse = __frcp_rn(scale);
    uint2* to = reinterpret_cast<uint2*>(codes + (uint64_t)held * p.head_dim);
    for (uint32_t base = threadIdx.x; base < vectors; base += kThreads * kMost) {
#pragma unroll
        for (uint32_t k = 0; k < kMost; ++k) {
            const uint32_t i = base + k * kThreads;
            if (i >= vectors) break;
            if (!once) x[k].load(at(i));
            float f[8];
            x[k].floats(f);
            if (odd) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = f[e] == f[e] ? f[e] : 0.0f;
            }
            to[i] = make_uint2(q8x4_quot(f[0], f[1], f[2], f[3], scale, inverse),
                               q8x4_quot(f[4], f[5], f[6], f[7], scale, inverse));
        }
    }
    __syncthreads();  // every thread has read the old scale
    if (grows && threadIdx.x == 0) p.scales[which][unit] = scale;
}

template <uint32_t kThreads>
void start(const AppendParams& p, uint32_t blocks, uint32_t precision, cudaStream_t st) {
    if (precision == 0) kv_cache_append_kernel<float, kThreads><<<blocks, kThreads, 0, st>>>(p);
    else if (precision == 1) kv_cache_append_kernel<__nv_bfloat16, kThreads><<<blocks, kThreads, 0, st>>>(p);
    else kv_cache_append_kernel<__half, kThreads><<<blocks, kThreads, 0, st>>>(p);
}

}  // namespace
}  // namespace dav2cuda

using namespace dav2cuda;

extern "C" DAV2CUDA_API int dav2cuda_kv_cache_append_s8(
    int8_t* k_codes, float* k_scales, int8_t* v_codes, float* v_scales, const void* k, const void* v,
    const int32_t* page_table, const int32_t* cached, const int32_t* token_begin, uint32_t sequences, uint32_t tokens,
    uint32_t kv_heads, uint32_t head_dim, uint32_t page_count, uint32_t page_tokens, uint32_t table_stride,
    uint64_t k_stride, uint64_t v_stride, uint32_t precision, void* stream) {
    DAV2_REQUIRE(precision <= 2, "cache append: unknown precision");
    DAV2_REQUIRE(head_dim >= 16 && head_dim <= 128 && head_dim % 16 == 0,
                 "cache append: head_dim must be a multiple of 16, 16 to 128");
    DAV2_REQUIRE(page_tokens >= 16 && page_tokens <= 128 && (page_tokens & (page_tokens - 1)) == 0,
                 "cache append: page_tokens must be 16, 32, 64 or 128");
    DAV2_REQUIRE(kv_heads >= 1 && kv_heads <= 32767 && page_count >= 1 && page_count <= 0x7FFFFFFFu && table_stride >= 1,
                 "invalid cache append dimensions");
    DAV2_REQUIRE(tokens <= 0x7FFFFFFFu && sequences <= 0x1FFFFFFFu, "cache append: too many tokens or sequences");
    if (tokens == 0 || sequences == 0) return DAV2CUDA_OK;
    const uint64_t row = (uint64_t)kv_heads * head_dim;
    DAV2_REQUIRE(tokens == 1 || (k_stride >= row && v_stride >= row),
                 "cache append: a token stride is below the row of its heads");
    DAV2_REQUIRE(!any_null(k_codes, k_scales, v_codes, v_scales, k, v, page_table, cached, token_begin),
                 "cache append: null buffer");
    const uint64_t bytes = element_bytes(precision);
    DAV2_REQUIRE(aligned16(k_codes) && aligned16(v_codes) && aligned16(k) && aligned16(v) &&
                     (tokens == 1 || (k_stride * bytes % 16 == 0 && v_stride * bytes % 16 == 0)),
                 "cache append: codes and rows must be 16-byte aligned");
    AppendParams p;
    p.codes[0] = k_codes, p.codes[1] = v_codes;
    p.scales[0] = k_scales, p.scales[1] = v_scales;
    p.rows[0] = k, p.rows[1] = v;
    p.stride[0] = k_stride, p.stride[1] = v_stride;
    p.page_table = page_table, p.cached = cached, p.begin = token_begin;
    p.sequences = sequences, p.tokens = tokens, p.heads = kv_heads, p.head_dim = head_dim, p.pages = page_count;
    p.page_shift = 4;
    while ((1u << p.page_shift) < page_tokens) ++p.page_shift;
    p.table_stride = table_stride;
    p.err = device_error_word();
    if (!p.err) return set_error(DAV2CUDA_INTERNAL_ERROR, "cache append: no device error word");
    const uint64_t blocks = ((uint64_t)(tokens >> p.page_shift) + 2ull * sequences) * kv_heads * 2;
    DAV2_REQUIRE(blocks <= 0x7FFFFFFFu, "cache append: too many tokens or sequences");
    const cudaStream_t st = as_stream(stream);
    // a few tokens for each sequence are the work of few threads, and blocks of few threads all
    // fit the SMs at once (64 sequences, one token each: 5.9 us, with 128 threads 7.4)
    if (tokens <= 4ull * sequences) start<64>(p, (uint32_t)blocks, precision, st);
    else start<128>(p, (uint32_t)blocks, precision, st);
    return check_launch("kv_cache_append_s8");
}

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
// Bound by memory: the rows are read from HBM once (the second pass over a
// page's rows, at most 128 rows of one head, finds them in L1 or L2) and the codes
// written once. One block for each page that receives tokens, each head, and K or
// V; the blocks of sequence s are numbered from floor(begin[s] / page_tokens) + 2 s,
// which leaves room for its pages whatever their boundaries, so that the host
// needs no length: blocks without a page leave at once.
#include "abi_check.h"
#include "kernels.cuh"

namespace dav2cuda {
namespace {

constexpr uint32_t kThreads = 128;

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

// Eight consecutive values as f32; NaN as 0.
template <typename T>
__device__ __forceinline__ void load8(float (&x)[8], const T* p) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        union {
            uint4 u;
            T t[8];
        } a;
        a.u = *reinterpret_cast<const uint4*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(a.t[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] == x[i] ? x[i] : 0.0f;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) kv_cache_append_kernel(const AppendParams p) {
    const uint32_t which = blockIdx.z, head = blockIdx.y;
    const uint32_t page_tokens = 1u << p.page_shift;
    // the last sequence whose blocks begin at or before this one
    const uint32_t s = warp_last_at_most(p.sequences, blockIdx.x, [&](uint32_t i) {
        return (uint64_t)((uint32_t)p.begin[i] >> p.page_shift) + 2 * i;
    });
    const int64_t begin = p.begin[s], end = p.begin[s + 1], cached = p.cached[s];
    const int64_t j = (int64_t)blockIdx.x - ((begin >> p.page_shift) + 2 * (int64_t)s);
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

    float most = 0.0f;
    for (uint32_t i = threadIdx.x; i < count * per_row; i += kThreads) {
        const uint32_t row = i / per_row, col = i - row * per_row;
        float x[8];
        load8(x, rows + row * p.stride[which] + col * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = fabsf(x[e]);
            most = fmaxf(most, a < INFINITY ? a : 0.0f);
        }
    }
    __shared__ float s_most[kThreads / 32];
    most = warp_max(most);
    if ((threadIdx.x & 31) == 0) s_most[threadIdx.x / 32] = most;
    const float old = held ? p.scales[which][unit] : 0.0f;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 32; ++w) most = fmaxf(most, s_most[w]);
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
    for (uint32_t i = threadIdx.x; i < count * per_row; i += kThreads) {
        const uint32_t row = i / per_row, col = i - row * per_row;
        float x[8];
        load8(x, rows + row * p.stride[which] + col * 8);
        to[i] = make_uint2(q8x4_quot(x[0], x[1], x[2], x[3], scale, inverse),
                           q8x4_quot(x[4], x[5], x[6], x[7], scale, inverse));
    }
    __syncthreads();  // every thread has read the old scale
    if (grows && threadIdx.x == 0) p.scales[which][unit] = scale;
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
    DAV2_REQUIRE(kv_heads >= 1 && kv_heads <= 65535 && page_count >= 1 && page_count <= 0x7FFFFFFFu && table_stride >= 1,
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
    const dim3 grid((tokens >> p.page_shift) + 2 * sequences, kv_heads, 2);
    const cudaStream_t st = as_stream(stream);
    if (precision == 0) kv_cache_append_kernel<float><<<grid, kThreads, 0, st>>>(p);
    else if (precision == 1) kv_cache_append_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(p);
    else kv_cache_append_kernel<__half><<<grid, kThreads, 0, st>>>(p);
    return check_launch("kv_cache_append_s8");
}

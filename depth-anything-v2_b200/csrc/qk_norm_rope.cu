// Queries and keys of an attention layer: a norm over each head and the
// rotation by position, in one pass over the rows.
//
//   y = x | x * rsqrt(mean(x^2) + eps) * w + b | (x - mean) * rsqrt(var + eps) * w + b
//   (u, v) -> s * (u cos a - v sin a, v cos a + u sin a), a = position * frequency
//
// on each pair (u, v) of the rotary part; the rest of the head keeps y.
//
// Bound by memory: x is read once and y written once; statistics and rotation
// are done on f32 values in registers. A block takes a few tokens and all (or,
// with few tokens, some) of their heads. It first puts the cosines and sines of
// its tokens' pairs and the norm's weights into shared memory, so that an angle
// is computed once for all heads; then a group of lanes takes a head at a time,
// each lane holding two vectors of V values that are the two halves of V pairs
// (interleaved pairs: 2V consecutive values). V is 8 where sizes, strides and
// addresses allow 16-byte accesses and 1 otherwise.
//
// 10960 tokens x 32 heads of 64, f32 to f16, in 27 us (4.9 TB/s); 32768 tokens x 40 heads of
// 128, bf16, in 109 us (6.2 TB/s). Three tokens take 3.1 us, nearly all of it a launch and
// three dependent accesses (frequencies and weights, rows, the sum over the lanes).
//
// An angle is position * frequency reduced by whole turns in 64 bits: in f32 it
// would be off by position * 2^-24 radians, 0.06 at a million tokens.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "abi_check.h"
#include "kernels.cuh"

namespace dav2cuda {
namespace {

constexpr uint32_t kMaxHead = 256;
constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxTokens = 8;  // tokens of one block

struct RopeParams {
    void* out[2];  // q, k
    const void* in[2];
    const float* weight[2];
    const float* bias[2];
    const float* frequencies;
    const int32_t* positions;
    uint64_t in_stride[2], out_stride[2];  // elements between tokens
    uint32_t heads[2];
    uint32_t tokens, head_dim, rotary, axes, layout, norm, block_tokens, head_splits;
    float epsilon, rotary_scale;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

template <typename T, int V>
__device__ __forceinline__ void load_vec(float (&x)[V], const T* p) {
    if constexpr (V == 1) {
        x[0] = to_f32(*p);
    } else {
        union {
            uint4 u[V * sizeof(T) / 16];
            T t[V];
        } a;
#pragma unroll
        for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) a.u[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = to_f32(a.t[i]);
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[V]) {
    if constexpr (V == 1) {
        *p = from_f32<T>(x[0]);
    } else {
        union {
            uint4 u[V * sizeof(T) / 16];
            T t[V];
        } a;
#pragma unroll
        for (int i = 0; i < V; ++i) a.t[i] = from_f32<T>(x[i]);
#pragma unroll
        for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) reinterpret_cast<uint4*>(p)[i] = a.u[i];
    }
}

template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const RopeParams p) {
    constexpr uint32_t U = V == 1 ? kMaxHead / 2 / 32 : 1;  // pair vectors of one lane
    __shared__ float s_cos[kMaxTokens * kMaxHead / 2], s_sin[kMaxTokens * kMaxHead / 2];
    __shared__ float s_weight[2][kMaxHead], s_bias[2][kMaxHead];
    const uint32_t pairs = p.rotary / 2, per_axis = pairs ? pairs / p.axes : 1;
    const uint32_t token0 = blockIdx.x * p.block_tokens;
    const uint32_t tokens = min(p.block_tokens, p.tokens - token0);

    for (uint32_t i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const uint32_t t = i / pairs, j = i - t * pairs;
        const uint32_t token = token0 + t;
        const double position =
            p.positions ? (double)p.positions[(uint64_t)token * p.axes + j / per_axis] : (double)token;
        const double half_turns = position * (double)p.frequencies[j] * 0.31830988618379067154;
        float sine, cosine;
        sincospif((float)(half_turns - 2.0 * rint(0.5 * half_turns)), &sine, &cosine);
        s_cos[i] = cosine * p.rotary_scale;
        s_sin[i] = sine * p.rotary_scale;
    }
    if (p.norm) {
        for (uint32_t i = threadIdx.x; i < 2 * p.head_dim; i += kThreads) {
            const uint32_t which = i >= p.head_dim, d = i - which * p.head_dim;
            s_weight[which][d] = p.weight[which] ? p.weight[which][d] : 1.0f;
            s_bias[which][d] = p.bias[which] ? p.bias[which][d] : 0.0f;
        }
    }
    __syncthreads();

    const uint32_t units = p.head_dim / (2 * V);
    uint32_t lanes = 32;  // lanes of one head
    if constexpr (V != 1) {
        lanes = 1;
        while (lanes < units) lanes *= 2;
    }
    const uint32_t lane = threadIdx.x & (lanes - 1);
    const uint32_t groups = kThreads / lanes, group = threadIdx.x / lanes;
    const uint32_t heads = p.heads[0] + p.heads[1];
    const uint32_t part = (heads + p.head_splits - 1) / p.head_splits;
    const uint32_t head0 = blockIdx.y * part, my_heads = head0 < heads ? min(part, heads - head0) : 0;

    // the places of this lane's vectors in a head
    uint32_t at0[U], at1[U];
#pragma unroll
    for (uint32_t k = 0; k < U; ++k) {
        const uint32_t j = (lane + 32 * k) * V;  // the first pair
        if (j < pairs) {
            const uint32_t axis = p.layout == 2 ? j / per_axis : 0;
            const uint32_t span = p.layout == 2 ? per_axis : pairs;
            at0[k] = p.layout == 1 ? 2 * j : j + axis * per_axis;
            at1[k] = p.layout == 1 ? 2 * j + V : at0[k] + span;
        } else {
            at0[k] = 2 * j;
            at1[k] = 2 * j + V;
        }
    }
    const uint32_t rows = tokens * my_heads;
    // every lane of a warp runs as often as the others: the shuffles need them all
    for (uint32_t base = 0; base < rows; base += groups) {
        const uint32_t r = base + group;
        const bool row_live = r < rows;
        const uint32_t t = row_live ? r / my_heads : 0;
        const uint32_t head = head0 + (row_live ? r - t * my_heads : 0);
        const uint32_t which = head >= p.heads[0];
        const uint32_t h = which ? head - p.heads[0] : head;
        const uint64_t token = token0 + t;
        const TI* in = static_cast<const TI*>(p.in[which]) + token * p.in_stride[which] + (uint64_t)h * p.head_dim;
        TO* out = static_cast<TO*>(p.out[which]) + token * p.out_stride[which] + (uint64_t)h * p.head_dim;
        float u[U][V], v[U][V];
#pragma unroll
        for (uint32_t k = 0; k < U; ++k) {
            if (row_live && lane + 32 * k < units) {
                load_vec<TI, V>(u[k], in + at0[k]);
                load_vec<TI, V>(v[k], in + at1[k]);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) u[k][i] = v[k][i] = 0.0f;
            }
        }
        if (p.norm) {
            const float inv_dim = 1.0f / (float)p.head_dim;
            if (p.norm == 2) {
                float sum = 0.0f;
#pragma unroll
                for (uint32_t k = 0; k < U; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) sum += u[k][i] + v[k][i];
                for (uint32_t o = lanes / 2; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const float mean = sum * inv_dim;
#pragma unroll
                for (uint32_t k = 0; k < U; ++k)
                    if (lane + 32 * k < units) {
#pragma unroll
                        for (int i = 0; i < V; ++i) u[k][i] -= mean, v[k][i] -= mean;
                    }
            }
            float sum = 0.0f;
#pragma unroll
            for (uint32_t k = 0; k < U; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) sum = fmaf(u[k][i], u[k][i], fmaf(v[k][i], v[k][i], sum));
            for (uint32_t o = lanes / 2; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float r_std = rsqrtf(sum * inv_dim + p.epsilon);
#pragma unroll
            for (uint32_t k = 0; k < U; ++k)
                if (lane + 32 * k < units) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        u[k][i] = fmaf(u[k][i] * r_std, s_weight[which][at0[k] + i], s_bias[which][at0[k] + i]);
                        v[k][i] = fmaf(v[k][i] * r_std, s_weight[which][at1[k] + i], s_bias[which][at1[k] + i]);
                    }
                }
        }
#pragma unroll
        for (uint32_t k = 0; k < U; ++k) {
            const uint32_t j = (lane + 32 * k) * V;
            if (j >= pairs) continue;
            const float* c = s_cos + t * pairs + j;
            const float* s = s_sin + t * pairs + j;
            if (p.layout == 1 && V > 1) {
                // 2V consecutive values: pair i lies at places 2i and 2i + 1
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const float a = u[k][2 * i], b = u[k][2 * i + 1], e = v[k][2 * i], f = v[k][2 * i + 1];
                    u[k][2 * i] = a * c[i] - b * s[i];
                    u[k][2 * i + 1] = b * c[i] + a * s[i];
                    v[k][2 * i] = e * c[V / 2 + i] - f * s[V / 2 + i];
                    v[k][2 * i + 1] = f * c[V / 2 + i] + e * s[V / 2 + i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float a = u[k][i], b = v[k][i];
                    u[k][i] = a * c[i] - b * s[i];
                    v[k][i] = b * c[i] + a * s[i];
                }
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < U; ++k)
            if (row_live && lane + 32 * k < units) {
                store_vec<TO, V>(out + at0[k], u[k]);
                store_vec<TO, V>(out + at1[k], v[k]);
            }
    }
}

template <typename TI, typename TO>
int launch(const RopeParams& p, bool vectors, cudaStream_t st) {
    const dim3 grid((p.tokens + p.block_tokens - 1) / p.block_tokens, p.head_splits);
    if (vectors) qk_norm_rope_kernel<TI, TO, 8><<<grid, kThreads, 0, st>>>(p);
    else qk_norm_rope_kernel<TI, TO, 1><<<grid, kThreads, 0, st>>>(p);
    return check_launch("qk_norm_rope");
}

}  // namespace
}  // namespace dav2cuda

using namespace dav2cuda;

extern "C" DAV2CUDA_API int dav2cuda_rope_frequencies(float* host_frequencies, float* host_rotary_scale,
                                                      uint32_t rotary_dim, uint32_t axes, double base,
                                                      uint32_t scaling, double factor, double trained_length) {
    DAV2_REQUIRE(!any_null(host_frequencies, host_rotary_scale), "rope frequencies: null buffer");
    DAV2_REQUIRE(rotary_dim && axes && rotary_dim % (2ull * axes) == 0 && rotary_dim <= kMaxHead,
                 "rope frequencies: rotary_dim must be a multiple of 2 * axes, at most 256");
    DAV2_REQUIRE(std::isfinite(base) && base > 1.0, "rope frequencies: base must be above 1");
    DAV2_REQUIRE(scaling <= 3, "rope frequencies: unknown scaling");
    DAV2_REQUIRE(scaling == 0 || (std::isfinite(factor) && factor >= 1.0),
                 "rope frequencies: factor must be 1 or more");
    DAV2_REQUIRE(scaling != 3 || (std::isfinite(trained_length) && trained_length > 0.0),
                 "rope frequencies: trained_length must be positive");
    const uint32_t count = rotary_dim / 2 / axes;
    if (scaling == 2 && count > 1) base *= std::pow(factor, (double)count / (count - 1));
    for (uint32_t j = 0; j < count; ++j) {
        double f = std::pow(base, -(double)j / count);
        if (scaling == 1) f /= factor;
        if (scaling == 3) {
            const double turns = trained_length * f / 6.283185307179586477;
            const double keep = std::fmin(std::fmax((turns - 1.0) / 31.0, 0.0), 1.0);
            f = f * keep + f / factor * (1.0 - keep);
        }
        for (uint32_t a = 0; a < axes; ++a) host_frequencies[a * count + j] = (float)f;
    }
    *host_rotary_scale = scaling == 3 ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return DAV2CUDA_OK;
}

extern "C" DAV2CUDA_API int dav2cuda_qk_norm_rope(
    void* q_output, void* k_output, const void* q, const void* k, const float* q_weight, const float* q_bias,
    const float* k_weight, const float* k_bias, const float* frequencies, const int32_t* positions, uint32_t tokens,
    uint32_t q_heads, uint32_t k_heads, uint32_t head_dim, uint32_t rotary_dim, uint32_t axes,
    uint64_t q_output_stride, uint64_t k_output_stride, uint64_t q_stride, uint64_t k_stride, uint32_t norm,
    float epsilon, uint32_t layout, float rotary_scale, uint32_t input_precision, uint32_t output_precision,
    void* stream) {
    DAV2_REQUIRE(head_dim >= 2 && head_dim <= kMaxHead && head_dim % 2 == 0,
                 "qk norm rope: head_dim must be even, 2 to 256");
    DAV2_REQUIRE(axes >= 1 && rotary_dim <= head_dim && rotary_dim % (2ull * axes) == 0,
                 "qk norm rope: rotary_dim must be a multiple of 2 * axes, at most head_dim");
    DAV2_REQUIRE(norm <= 2 && layout <= 2, "qk norm rope: unknown norm or layout");
    DAV2_REQUIRE(norm == 0 || (epsilon >= 0.0f && std::isfinite(epsilon)), "qk norm rope: invalid epsilon");
    DAV2_REQUIRE(std::isfinite(rotary_scale), "qk norm rope: invalid rotary scale");
    DAV2_REQUIRE(input_precision <= 2 && output_precision <= 2 &&
                     (input_precision == 0 || output_precision == input_precision),
                 "qk norm rope: output must be of the input's type (f32 input: any)");
    DAV2_REQUIRE((uint64_t)q_heads + k_heads > 0 && (uint64_t)q_heads + k_heads <= 65535,
                 "qk norm rope: 1 to 65535 heads");
    const uint64_t q_row = (uint64_t)q_heads * head_dim, k_row = (uint64_t)k_heads * head_dim;
    DAV2_REQUIRE(tokens <= 1 || ((q_stride >= q_row && q_output_stride >= q_row) || !q_heads),
                 "qk norm rope: a token stride is below the row of its heads");
    DAV2_REQUIRE(tokens <= 1 || ((k_stride >= k_row && k_output_stride >= k_row) || !k_heads),
                 "qk norm rope: a token stride is below the row of its heads");
    if (tokens == 0) return DAV2CUDA_OK;
    DAV2_REQUIRE((q_heads == 0 || !any_null(q_output, q)) && (k_heads == 0 || !any_null(k_output, k)) &&
                     (rotary_dim == 0 || frequencies),
                 "qk norm rope: null buffer");
    DAV2_REQUIRE(axes == 1 || rotary_dim == 0 || positions, "qk norm rope: several axes need positions");

    RopeParams p{};
    p.out[0] = q_output, p.out[1] = k_output;
    p.in[0] = q, p.in[1] = k;
    p.weight[0] = q_weight, p.weight[1] = k_weight;
    p.bias[0] = q_bias, p.bias[1] = k_bias;
    p.frequencies = frequencies, p.positions = positions;
    p.in_stride[0] = q_stride, p.in_stride[1] = k_stride;
    p.out_stride[0] = q_output_stride, p.out_stride[1] = k_output_stride;
    p.heads[0] = q_heads, p.heads[1] = k_heads;
    p.tokens = tokens, p.head_dim = head_dim, p.rotary = rotary_dim, p.axes = axes;
    p.layout = layout, p.norm = norm, p.epsilon = epsilon, p.rotary_scale = rotary_scale;

    const uint32_t per_axis = rotary_dim / 2 / axes;
    bool vectors = head_dim % 16 == 0 && rotary_dim % 16 == 0 && (layout != 2 || per_axis % 8 == 0);
    for (int w = 0; w < 2; ++w) {
        if (!p.heads[w]) continue;
        const uint32_t in_step = 16 / element_bytes(input_precision), out_step = 16 / element_bytes(output_precision);
        vectors = vectors && aligned16(p.in[w]) && aligned16(p.out[w]);
        vectors = vectors && (tokens == 1 || (p.in_stride[w] % in_step == 0 && p.out_stride[w] % out_step == 0));
    }
    int dev = 0;
    cudaGetDevice(&dev);
    const uint32_t sms = (uint32_t)sm_count(dev);
    if (!sms) return set_error(DAV2CUDA_LAUNCH_FAILED, "qk norm rope: cannot query the SM count");
    // Eight tokens to a block, so that a block's angles serve many rows; one token,
    // and its heads over several blocks, where that would leave SMs idle.
    const uint32_t heads = q_heads + k_heads;
    p.block_tokens = tokens >= 16 * sms ? kMaxTokens : 1;
    uint32_t lanes = 32;
    if (vectors)
        for (lanes = 1; lanes < head_dim / 16;) lanes *= 2;
    const uint32_t groups = kThreads / lanes, most = (heads + groups - 1) / groups;
    p.head_splits = p.block_tokens > 1 ? 1 : std::min(most, (2 * sms + tokens - 1) / tokens);

    const cudaStream_t st = as_stream(stream);
    if (input_precision == 1) return launch<__nv_bfloat16, __nv_bfloat16>(p, vectors, st);
    if (input_precision == 2) return launch<__half, __half>(p, vectors, st);
    if (output_precision == 1) return launch<float, __nv_bfloat16>(p, vectors, st);
    if (output_precision == 2) return launch<float, __half>(p, vectors, st);
    return launch<float, float>(p, vectors, st);
}

// Entries of the grouped-head attention: cache of int8 codes, 16-bit cross
// attention. They check their arguments, choose the kernel and the splits, and launch.
#include <algorithm>
#include <cmath>

#include "abi_check.h"
#include "attention_rows.cuh"

namespace dav2cuda {
namespace {

// Plans are made for 148 SMs, a B200's, so that workspace sizes need no device.
constexpr uint32_t kSms = 148;

struct Plan {
    uint32_t row_tiles;  // 8-row tiles of a warp (rows kernel)
    uint32_t row_warps;  // row tiles of a block (rows kernel); 0: the tiles kernel
    uint32_t splits;     // of the keys
    bool clusters;       // whose splits join in a cluster, not in the workspace
    uint64_t slots;      // row blocks over all sequences
};

// The rows that share a key head, of a sequence on average, decide the kernel for the whole
// call: the host does not know the sequences' own. Keys are split where the row blocks
// alone would leave SMs idle, down to 128 keys (tiles kernel: 512) to a block.
Plan plan_rows(uint64_t sequences, uint64_t queries, bool s8, uint32_t max_length, uint32_t group,
               uint32_t kv_heads, uint32_t head_dim) {
    const bool ragged = s8;  // query_begin gives the rows of a sequence
    Plan n;
    const uint64_t each = ragged ? (queries + sequences - 1) / sequences : queries;
    const uint64_t rows = each * group;
    n.row_tiles = rows <= 8 ? 1 : 2;
    n.row_warps = rows <= 16 ? 1 : 2;
    // 16 sequences of 16 key heads, 32 and 64 rows of 64 dims over 2000 keys, rows and tiles kernel: 38.5 and
    // 54.0, 74.3 and 54.0 us; 8 caches of about 4000 tokens, 8 key heads, 64 rows of 128 dims: 82 and 51 us
    if (rows > 32) n.row_warps = 0;
    const uint64_t tile = n.row_warps ? 8ull * n.row_tiles * n.row_warps : 256;
    n.slots = ragged ? queries * group / tile + sequences : sequences * ((rows + tile - 1) / tile);
    const uint64_t live = std::max<uint64_t>(1, sequences * ((rows + tile - 1) / tile)) * kv_heads;
    n.clusters = false;
    if (!n.row_warps) {
        // the split count that ends first: rounds of units over the SMs, each a number of
        // 128-key blocks (about 2 us) and as much as eight more to begin and end; the parts, written
        // and read again, about 2 us for 5 MB, and the join a launch
        const uint64_t blocks = (max_length + 127ull) / 128;
        const uint64_t part = rows * sequences * kv_heads * (head_dim * 8ull + 16);
        uint64_t best = ~0ull;
        n.splits = 1;
        for (uint64_t s = 1; s <= 32 && s * 4 <= std::max<uint64_t>(blocks, 4); ++s) {
            const uint64_t cost = (live * s + kSms - 1) / kSms * ((blocks + s - 1) / s + 8) +
                                  (s > 1 ? 3 + s * part / 5000000 : 0);
            if (cost < best) best = cost, n.splits = (uint32_t)s;
        }
        // warps that are done with a unit wait for the next one, and a wait ends with an error after 4 s
        // (kWaitTimeoutNs): no unit is longer than 2^19 key blocks, under 2 s of 2 to 3.4 us each
        n.splits = std::max(n.splits, (uint32_t)((blocks + (1u << 19) - 1) >> 19));
        return n;
    }
    // The rows kernel. What fits the device at once is filled by one wave of equal
    // splits; where lengths may differ and are long, about two waves even out the end
    // (48 streams of up to 8192 keys: 1, 2, 3 splits 123, 110, 113 us). Up to eight
    // splits are a cluster and join there, without the workspace and a second launch.
    const uint64_t fit = (uint64_t)kSms * (s8 ? (head_dim <= 64 ? 6 : 3) : 2);
    const uint64_t most = std::max<uint64_t>(1, max_length / 128);
    uint64_t splits = std::max<uint64_t>(1, fit / live);
    if (sequences > 1) splits = std::max(splits, std::min<uint64_t>((2 * fit + live - 1) / live, max_length / 4096));
    if (splits > 8 && (live * 8 >= fit || max_length <= 4096)) splits = 8;
    n.splits = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(splits, most), kMaxSplits);
    n.clusters = n.splits > 1 && n.splits <= 8;
    return n;
}

uint64_t workspace_of(const Plan& n, uint64_t tokens, uint32_t heads, uint32_t head_dim) {
    if (n.splits == 1 || n.clusters) return 0;
    return tokens * heads * n.splits * (head_dim * 4ull + 8) + 256;
}

int run(RowsParams& p, const Plan& n, bool s8, bool bf16, uint64_t tokens, void* workspace, cudaStream_t st) {
    p.row_warps = n.row_warps, p.splits = n.splits, p.clusters = n.clusters;
    const uint64_t rows = tokens * p.kv_heads * p.group;
    const bool parts = n.splits > 1 && !n.clusters;
    if (parts) {
        uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 15) & ~uintptr_t(15));
        p.part_o = reinterpret_cast<float*>(base);
        p.part_ml = reinterpret_cast<float2*>(base + rows * n.splits * p.head_dim * 4);
    }
    if (int rc = n.row_warps ? launch_attention_rows(p, (uint32_t)n.slots, n.row_tiles, s8, bf16, st)
                             : launch_attention_tiles(p, (uint32_t)n.slots, s8, bf16, st))
        return rc;
    return parts ? launch_attention_join(p, rows, st) : DAV2CUDA_OK;
}

bool shape_ok(uint32_t q_heads, uint32_t kv_heads) {
    return q_heads >= 1 && kv_heads >= 1 && kv_heads <= 65535 && q_heads % kv_heads == 0 && q_heads <= 65535;
}

}  // namespace
}  // namespace dav2cuda

using namespace dav2cuda;

extern "C" DAV2CUDA_API uint64_t dav2cuda_attention_cache_s8_workspace_size(uint32_t sequences, uint32_t queries,
                                                                            uint32_t max_length, uint32_t q_heads,
                                                                            uint32_t kv_heads, uint32_t head_dim) {
    if (!sequences || !queries || !shape_ok(q_heads, kv_heads)) return 0;
    const Plan n = plan_rows(sequences, queries, true, max_length, q_heads / kv_heads, kv_heads, head_dim);
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
    const Plan n = plan_rows(sequences, queries, true, max_length, p.group, kv_heads, head_dim);
    DAV2_REQUIRE(n.slots <= 0x7FFFFFFFu, "cache attention: too many queries or sequences");
    const uint64_t need = workspace_of(n, queries, q_heads, head_dim);
    DAV2_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "cache attention: workspace is too small");
    p.err = device_error_word();
    if (!p.err) return set_error(DAV2CUDA_INTERNAL_ERROR, "cache attention: no device error word");
    return run(p, n, true, false, queries, workspace, as_stream(stream));
}

extern "C" DAV2CUDA_API uint64_t dav2cuda_cross_attention_16_workspace_size(uint32_t batch, uint32_t queries,
                                                                            uint32_t keys, uint32_t q_heads,
                                                                            uint32_t kv_heads, uint32_t head_dim) {
    if (!batch || !queries || !shape_ok(q_heads, kv_heads)) return 0;
    const Plan n = plan_rows(batch, queries, false, keys, q_heads / kv_heads, kv_heads, head_dim);
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
    // batch after batch, or (tokens first) the batches of a token one after another
    DAV2_REQUIRE(batch == 1 || output_batch_stride >= (queries - 1) * output_stride + row ||
                     (output_batch_stride >= row && output_stride >= (batch - 1) * output_batch_stride + row),
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
    const Plan n = plan_rows(batch, queries, false, keys, p.group, kv_heads, head_dim);
    DAV2_REQUIRE(n.slots <= 0x7FFFFFFFu, "cross attention: too many queries");
    const uint64_t tokens = (uint64_t)batch * queries, need = workspace_of(n, tokens, q_heads, head_dim);
    DAV2_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "cross attention: workspace is too small");
    p.err = device_error_word();
    if (!p.err) return set_error(DAV2CUDA_INTERNAL_ERROR, "cross attention: no device error word");
    return run(p, n, false, precision == 1, tokens, workspace, as_stream(stream));
}

// capi_kv8.cpp -- the 8-bit KV cache's part of the extern "C" surface (include/nvllm_attn.h):
// argument checks in front of the launchers of kv8_write.hip and paged_attn_kv8.hip.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/nvllm_attn.h"
#include "nvllm_host.hpp"
#include "nvllm_kernels.hpp"

using nvllm::ErrorKind;
namespace kernels = nvllm::kernels;

namespace {

int fail(ErrorKind kind, const char *who, const char *msg) {
    nvllm::set_last_error(kind, std::string(who) + ": " + msg);
    return static_cast<int>(kind);
}

int hip_status(hipError_t err, const char *who) {
    if (err == hipSuccess) return NVLLM_OK;
    return fail(ErrorKind::Hip, who, hipGetErrorString(err));
}

hipStream_t as_stream(nvllm_stream_t s) { return reinterpret_cast<hipStream_t>(s); }

bool aligned(const void *p, unsigned n) { return (reinterpret_cast<std::uintptr_t>(p) & (n - 1)) == 0; }

bool overlap(const void *a, std::int64_t a_bytes, const void *b, std::int64_t b_bytes) {
    const auto x = reinterpret_cast<std::uintptr_t>(a), y = reinterpret_cast<std::uintptr_t>(b);
    return x < y + (std::uintptr_t)b_bytes && y < x + (std::uintptr_t)a_bytes;
}

// what every entry on the cache checks: its geometry, the formats, the scales' alignment
int check_cache(const char *who, std::int64_t num_cache_blocks, int block_size, int num_kv_heads, int head_dim,
                int format, int dtype) {
    if (num_cache_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0 || head_dim <= 0)
        return fail(ErrorKind::Config, who, "negative or zero dimension");
    if (format != 0 && format != 1) return fail(ErrorKind::Unsupported, who, "format must be 0 (int8) or 1 (E4M3)");
    if (dtype != 0 && dtype != 1) return fail(ErrorKind::Unsupported, who, "dtype must be 0 (bf16) or 1 (f32)");
    if (head_dim > 256) return fail(ErrorKind::Unsupported, who, "head_dim > 256");
    if (num_cache_blocks > 0x7fffffff) return fail(ErrorKind::Unsupported, who, "more than 2^31 - 1 blocks");
    if (block_size > kernels::kKv8MaxBlockSize) return fail(ErrorKind::Unsupported, who, "block_size > 256");
    if ((int64_t)block_size * num_kv_heads * head_dim > 0x7fffffffLL)
        return fail(ErrorKind::Unsupported, who, "block of more than 2^31 - 1 values");
    return NVLLM_OK;
}

// what the writers count in 32 bits: tokens, and the pairs of block and head of 16 blocks
int check_writer(const char *who, std::int64_t num_tokens, int num_heads, int num_kv_heads) {
    if (num_heads > 65535 || num_kv_heads > 65535) return fail(ErrorKind::Unsupported, who, "more than 65535 heads");
    if (num_tokens > (1 << 30)) return fail(ErrorKind::Unsupported, who, "more than 2^30 tokens");
    return NVLLM_OK;
}

int write_common(const char *who, const kernels::Kv8WriteArgs &a, size_t workspace_bytes, int format, int dtype,
                 nvllm_stream_t stream) {
    if (!a.key || !a.value || !a.k_cache || !a.v_cache || !a.k_scales || !a.v_scales || !a.slot_mapping)
        return fail(ErrorKind::Null, who, "null pointer");
    const unsigned elt = dtype == 0 ? 2 : 4;
    if (!aligned(a.key, elt) || !aligned(a.value, elt) || !aligned(a.k_scales, 4) || !aligned(a.v_scales, 4) ||
        !aligned(a.slot_mapping, 8))
        return fail(ErrorKind::Config, who, "pointer not aligned to its element type");
    const size_t need = kernels::kv8_write_workspace_bytes(a.num_tokens, a.block_size, a.num_cache_blocks);
    if (need > 0 && (!a.workspace || workspace_bytes < need)) {
        nvllm::set_last_error(ErrorKind::Config,
                              std::string(who) + ": workspace of " + std::to_string(a.workspace ? workspace_bytes : 0) +
                                  " bytes, this call needs " + std::to_string(need) +
                                  " (nvllm_kv8_write_workspace_bytes)");
        return NVLLM_ERR_CONFIG;
    }
    if (need > 0 && !aligned(a.workspace, 16))
        return fail(ErrorKind::Config, who, "workspace must be 16-byte aligned");
    // K and V of a block are written by different waves
    const std::int64_t scales = a.num_cache_blocks * a.num_kv_heads * 4, codes = scales / 4 * a.block_size * a.head_dim;
    if (overlap(a.k_cache, codes, a.v_cache, codes) || overlap(a.k_scales, scales, a.v_scales, scales))
        return fail(ErrorKind::Config, who, "caches of K and V must not overlap, nor their scales");
    return hip_status(kernels::launch_kv8_write(static_cast<kernels::DType>(dtype),
                                                static_cast<kernels::Kv8Format>(format), a, as_stream(stream)),
                      who);
}

}  // namespace

extern "C" {

size_t nvllm_kv8_write_workspace_bytes(int64_t num_tokens, int block_size, int64_t num_cache_blocks) {
    if (num_tokens <= 0 || block_size <= 0 || num_cache_blocks <= 0) return 0;
    return kernels::kv8_write_workspace_bytes(num_tokens, block_size, num_cache_blocks);
}

int nvllm_reshape_and_cache_kv8(const void *key, const void *value, void *k_cache, void *v_cache, float *k_scales,
                                float *v_scales, const int64_t *slot_mapping, void *workspace,
                                size_t workspace_bytes, int64_t num_tokens, int num_kv_heads, int head_dim,
                                int block_size, int64_t num_cache_blocks, int format, int dtype,
                                nvllm_stream_t stream) {
    static const char *who = "reshape_and_cache_kv8";
    if (num_tokens < 0) return fail(ErrorKind::Config, who, "negative or zero dimension");
    if (const int rc = check_cache(who, num_cache_blocks, block_size, num_kv_heads, head_dim, format, dtype)) return rc;
    if (const int rc = check_writer(who, num_tokens, 0, num_kv_heads)) return rc;
    if (num_tokens == 0) return NVLLM_OK;
    kernels::Kv8WriteArgs a{};
    a.key = key;
    a.value = value;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k_scales = k_scales;
    a.v_scales = v_scales;
    a.slot_mapping = slot_mapping;
    a.workspace = static_cast<int32_t *>(workspace);
    a.num_tokens = num_tokens;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.block_size = block_size;
    a.num_cache_blocks = num_cache_blocks;
    return write_common(who, a, workspace_bytes, format, dtype, stream);
}

int nvllm_qk_norm_rope_cache_kv8(const void *q, const void *k, const void *v, void *q_out, void *k_out,
                                 const void *q_weight, const void *k_weight, float eps, const void *cos_cache,
                                 const void *sin_cache, int64_t max_positions, const int32_t *positions,
                                 void *k_cache, void *v_cache, float *k_scales, float *v_scales,
                                 const int64_t *slot_mapping, void *workspace, size_t workspace_bytes,
                                 int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, int block_size,
                                 int64_t num_cache_blocks, int format, int dtype, nvllm_stream_t stream) {
    static const char *who = "qk_norm_rope_cache_kv8";
    if (num_tokens < 0 || num_heads <= 0 || max_positions <= 0 || max_positions > 0x7fffffff)
        return fail(ErrorKind::Config, who, "negative or zero dimension");
    if (const int rc = check_cache(who, num_cache_blocks, block_size, num_kv_heads, head_dim, format, dtype)) return rc;
    if (const int rc = check_writer(who, num_tokens, num_heads, num_kv_heads)) return rc;
    if (head_dim % 2 != 0)  // rope.rs:49 assert!(dim.is_multiple_of(2))
        return fail(ErrorKind::Config, who, "RoPE dimension must be even");
    if (num_tokens == 0) return NVLLM_OK;
    if (!q || !q_out || !q_weight || !k_weight || !cos_cache || !sin_cache || !positions)
        return fail(ErrorKind::Null, who, "null pointer");
    const unsigned elt = dtype == 0 ? 2 : 4;
    for (const void *p : {q, (const void *)q_out, (const void *)k_out, q_weight, k_weight, cos_cache, sin_cache})
        if (!aligned(p, elt)) return fail(ErrorKind::Config, who, "pointer not aligned to its element type");
    if (!aligned(positions, 4)) return fail(ErrorKind::Config, who, "pointer not aligned to its element type");
    // other waves read rows of q, k and v while these are written
    const int64_t kv_bytes = num_tokens * num_kv_heads * head_dim * elt, q_bytes = num_tokens * num_heads * head_dim * elt;
    for (const void *p : {k, v}) {
        if (p && k_out && overlap(k_out, kv_bytes, p, kv_bytes))
            return fail(ErrorKind::Config, who, "k_out must not overlap k or v");
        if (p && overlap(q_out, q_bytes, p, kv_bytes))
            return fail(ErrorKind::Config, who, "q_out must not overlap k or v");
    }
    if (q_out != q && overlap(q_out, q_bytes, q, q_bytes))
        return fail(ErrorKind::Config, who, "q_out must be q or not overlap it");
    if (k_out && (overlap(k_out, kv_bytes, q, q_bytes) || overlap(k_out, kv_bytes, q_out, q_bytes)))
        return fail(ErrorKind::Config, who, "k_out must not overlap q or q_out");
    kernels::Kv8WriteArgs a{};
    a.key = k;
    a.value = v;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k_scales = k_scales;
    a.v_scales = v_scales;
    a.slot_mapping = slot_mapping;
    a.workspace = static_cast<int32_t *>(workspace);
    a.num_tokens = num_tokens;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.block_size = block_size;
    a.num_cache_blocks = num_cache_blocks;
    a.q = q;
    a.q_out = q_out;
    a.k_out = k_out;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.eps = eps;
    a.cos_cache = cos_cache;
    a.sin_cache = sin_cache;
    a.max_positions = (int)max_positions;
    a.positions = positions;
    a.num_heads = num_heads;
    return write_common(who, a, workspace_bytes, format, dtype, stream);
}

int nvllm_gather_cache_blocks_kv8(const void *k_cache, const void *v_cache, const float *k_scales,
                                  const float *v_scales, const int32_t *block_ids, int64_t num_ids, void *k_out,
                                  void *v_out, int64_t num_cache_blocks, int block_size, int num_kv_heads,
                                  int head_dim, int format, int dtype, nvllm_stream_t stream) {
    static const char *who = "gather_cache_blocks_kv8";
    if (num_ids <= 0)  // kv_cache.rs:124-126
        return fail(ErrorKind::Config, who, "block_ids cannot be empty");
    if (num_ids > 0x7fffffff) return fail(ErrorKind::Unsupported, who, "more than 2^31 - 1 block_ids");
    if (const int rc = check_cache(who, num_cache_blocks, block_size, num_kv_heads, head_dim, format, dtype)) return rc;
    if (!k_cache || !k_scales || !block_ids || !k_out || (v_out && (!v_cache || !v_scales)))
        return fail(ErrorKind::Null, who, "null pointer");
    const unsigned elt = dtype == 0 ? 2 : 4;
    if (!aligned(k_out, elt) || !aligned(v_out, elt) || !aligned(k_scales, 4) || !aligned(v_scales, 4) ||
        !aligned(block_ids, 4))
        return fail(ErrorKind::Config, who, "pointer not aligned to its element type");
    return hip_status(kernels::launch_kv8_gather(static_cast<kernels::DType>(dtype),
                                                 static_cast<kernels::Kv8Format>(format), k_cache, v_cache, k_scales,
                                                 v_scales, block_ids, num_ids, k_out, v_out, num_cache_blocks,
                                                 block_size, num_kv_heads, head_dim, as_stream(stream)),
                      who);
}

static kernels::PagedAttnArgs attn_shape(int num_seqs, int num_new_tokens, int num_heads, int num_kv_heads,
                                         int head_dim, int block_size, int max_blocks_per_seq) {
    kernels::PagedAttnArgs a{};
    a.num_seqs = num_seqs;
    a.num_new_tokens = num_new_tokens;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.block_size = block_size;
    a.max_blocks_per_seq = max_blocks_per_seq;
    return a;
}

static int check_attn(const char *who, int num_seqs, int num_new_tokens, int num_heads, int num_kv_heads,
                      int block_size, int max_blocks_per_seq) {
    if (num_seqs < 0 || num_new_tokens <= 0 || num_heads <= 0)
        return fail(ErrorKind::Config, who, "negative or zero dimension");
    if (max_blocks_per_seq <= 0)  // paged.rs:133-137
        return fail(ErrorKind::Config, who, "BlockTable is empty - no blocks allocated");
    if (num_heads % num_kv_heads != 0)
        return fail(ErrorKind::Config, who, "num_heads must be a multiple of num_kv_heads");
    if (num_seqs > 65535) return fail(ErrorKind::Unsupported, who, "num_seqs > 65535 per launch");
    if (num_kv_heads > 65535) return fail(ErrorKind::Unsupported, who, "num_kv_heads > 65535");
    if ((int64_t)max_blocks_per_seq * block_size > (1 << 30))
        return fail(ErrorKind::Unsupported, who, "block tables of more than 2^30 tokens");
    if ((int64_t)num_heads * num_new_tokens > 0x7fffffffLL)
        return fail(ErrorKind::Unsupported, who, "more than 2^31 - 1 query rows per sequence");
    return NVLLM_OK;
}

size_t nvllm_paged_attn_kv8_workspace_bytes(int num_seqs, int num_new_tokens, int num_heads, int num_kv_heads,
                                            int head_dim, int block_size, int max_blocks_per_seq, int dtype) {
    if (num_seqs <= 0 || num_new_tokens <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
        block_size <= 0 || max_blocks_per_seq <= 0 || num_heads % num_kv_heads != 0 || (dtype != 0 && dtype != 1))
        return 0;
    return kernels::paged_attn_kv8_workspace_bytes(
        static_cast<kernels::DType>(dtype),
        attn_shape(num_seqs, num_new_tokens, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq));
}

int nvllm_paged_attn_kv8_path(int num_seqs, int num_new_tokens, int num_heads, int num_kv_heads, int head_dim,
                              int block_size, int max_blocks_per_seq, int dtype) {
    static const char *who = "paged_attn_kv8_path";
    if (const int rc = check_cache(who, 1, block_size, num_kv_heads, head_dim, 0, dtype)) return rc;
    if (const int rc = check_attn(who, num_seqs, num_new_tokens, num_heads, num_kv_heads, block_size,
                                  max_blocks_per_seq))
        return rc;
    return (int)kernels::paged_attn_kv8_path(
        static_cast<kernels::DType>(dtype),
        attn_shape(num_seqs, num_new_tokens, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq));
}

int nvllm_paged_attn_kv8(const void *q, const void *k_cache, const void *v_cache, const float *k_scales,
                         const float *v_scales, const int32_t *block_tables, const int32_t *context_lens, void *out,
                         void *workspace, size_t workspace_bytes, int num_seqs, int num_new_tokens, int num_heads,
                         int num_kv_heads, int head_dim, int block_size, int max_blocks_per_seq,
                         int64_t num_cache_blocks, float scale, int format, int dtype, nvllm_stream_t stream) {
    static const char *who = "paged_attn_kv8";
    if (const int rc = check_cache(who, num_cache_blocks, block_size, num_kv_heads, head_dim, format, dtype)) return rc;
    if (const int rc = check_attn(who, num_seqs, num_new_tokens, num_heads, num_kv_heads, block_size,
                                  max_blocks_per_seq))
        return rc;
    if (num_seqs == 0) return NVLLM_OK;
    if (!q || !k_cache || !v_cache || !k_scales || !v_scales || !block_tables || !context_lens || !out)
        return fail(ErrorKind::Null, who, "null pointer");
    const unsigned elt = dtype == 0 ? 2 : 4;
    if (!aligned(q, elt) || !aligned(out, elt) || !aligned(k_scales, 4) || !aligned(v_scales, 4) ||
        !aligned(block_tables, 4) || !aligned(context_lens, 4))
        return fail(ErrorKind::Config, who, "pointer not aligned to its element type");
    kernels::PagedAttnArgs a =
        attn_shape(num_seqs, num_new_tokens, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq);
    const kernels::DType dt = static_cast<kernels::DType>(dtype);
    if (kernels::paged_attn_kv8_path(dt, a) != kernels::PagedKv8Path::Generic &&
        !(aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16)))
        return fail(ErrorKind::Config, who, "tensors must be 16-byte aligned");
    const size_t need = kernels::paged_attn_kv8_workspace_bytes(dt, a);
    if (need > 0 && (!workspace || workspace_bytes < need)) {
        nvllm::set_last_error(ErrorKind::Config,
                              std::string(who) + ": workspace of " + std::to_string(workspace ? workspace_bytes : 0) +
                                  " bytes, this launch shape needs " + std::to_string(need) +
                                  " (nvllm_paged_attn_kv8_workspace_bytes)");
        return NVLLM_ERR_CONFIG;
    }
    if (need > 0 && !aligned(workspace, 16))
        return fail(ErrorKind::Config, who, "workspace must be 16-byte aligned");
    a.q = q;
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.block_tables = block_tables;
    a.context_lens = context_lens;
    a.out = out;
    a.workspace = need > 0 ? workspace : nullptr;
    a.workspace_bytes = need > 0 ? workspace_bytes : 0;
    a.num_cache_blocks = num_cache_blocks;
    a.scale = scale;
    return hip_status(kernels::launch_paged_attn_kv8(dt, static_cast<kernels::Kv8Format>(format), a, k_scales,
                                                     v_scales, as_stream(stream)),
                      who);
}

int64_t nvllm_kv_cache_kv8_layer_bytes(int64_t num_blocks, int64_t block_size, int64_t num_kv_heads,
                                       int64_t head_dim) {
    if (num_blocks < 0 || block_size < 0 || num_kv_heads < 0 || head_dim < 0) return -1;
    return num_blocks * num_kv_heads * (block_size * head_dim + 4);
}

}  // extern "C"

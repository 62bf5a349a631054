// paged_attn_kv8.hip -- paged attention over the 8-bit KV cache (gfx950).
//
// The block tables, context lengths and the bottom-right causal mask are those of paged_attn.hip
// (reference src/attention/paged.rs:117-192, :357-381); K and V are codes with one scale per (block,
// kv head), kv8_common.hpp:
//   s_ij = softmax_scale * kscale[block of j] * (q_i . kcode_j),   p_ij = exp(s_ij - max_j s_ij)
//   o_i  = sum_j (p_ij * vscale[block of j]) vcode_j / sum_j p_ij
// A scale belongs to a token (its block), so it multiplies scores and probabilities and never the
// codes: what is converted is one byte to the matrix unit's type, exactly.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "kv8_common.hpp"

namespace nvllm {
namespace kernels {

namespace {

using namespace kv8;

// ---------------------------------------------------------------------------
// Generic path: any head_dim <= 256, any block size, bf16 or f32.  One workgroup per (sequence, new
// token, query head); its four waves take every fourth tile of 64 keys and join at the end.  f32 FMA.
// A lane is a key for q.k and four dims for p.v.
// ---------------------------------------------------------------------------
template <typename ET, Kv8Format F>
__global__ __launch_bounds__(256) void paged_attn_kv8_generic_kernel(
    const ET *__restrict__ q, const unsigned char *__restrict__ k_cache, const unsigned char *__restrict__ v_cache,
    const float *__restrict__ k_scales, const float *__restrict__ v_scales, const int32_t *__restrict__ block_tables,
    const int32_t *__restrict__ context_lens, ET *__restrict__ out, int T, int Hq, int Hkv, int D, int block_size,
    int max_blocks_per_seq, int64_t num_cache_blocks, float scale, bool wide) {
    __shared__ float q_s[256];
    __shared__ float p_s[4][64];
    __shared__ int64_t row_s[4][64];  // element offset of each key's row
    __shared__ float o_s[4][256];
    __shared__ float m_s[4], l_s[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = (int)(blockIdx.x % (unsigned)Hq), t = (int)(blockIdx.x / (unsigned)Hq), seq = blockIdx.y;
    const int kvh = h / (Hq / Hkv);
    int64_t ctx = context_lens[seq];
    const int64_t cap = (int64_t)max_blocks_per_seq * block_size;
    if (ctx > cap) ctx = cap;  // never read past the table row
    const int64_t keys = ctx - T + t + 1;  // keys this query sees: 0 .. keys - 1 (none if <= 0)
    const int64_t orow = (((int64_t)seq * T + t) * Hq + h) * D;
    for (int d = threadIdx.x; d < 256; d += 256) {
        q_s[d] = d < D ? to_f32(q[orow + d]) : 0.0f;
        for (int w = 0; w < 4; ++w) o_s[w][d] = 0.0f;
    }
    __syncthreads();
    const int32_t *table = block_tables + (int64_t)seq * max_blocks_per_seq;
    const int lanes = wide ? D / 4 : 64, together = wide ? 64 / lanes : 1;  // lanes per V row, rows at once
    const int vr = wide ? lane / lanes : 0, vc = wide ? lane % lanes : lane;
    float m = -INFINITY, l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t base = 64 * wave; base < keys; base += 256) {
        const int64_t key = base + lane;
        float s = -INFINITY, vs = 0.0f;
        if (key < keys) {
            const int64_t lb = key / block_size;
            int64_t pb = table[lb];
            pb = pb < 0 ? 0 : (pb >= num_cache_blocks ? num_cache_blocks - 1 : pb);
            const int64_t row = ((pb * block_size + (key - lb * block_size)) * Hkv + kvh) * D;
            row_s[wave][lane] = row;
            float acc = 0.0f;
            if (wide) {
                for (int d = 0; d < D; d += 4) {
                    float x[4];
                    decode4<F>(*reinterpret_cast<const unsigned *>(k_cache + row + d), x);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc += q_s[d + i] * x[i];
                }
            } else {
                for (int d = 0; d < D; ++d) acc += q_s[d] * decode1<F>(k_cache[row + d]);
            }
            s = acc * (scale * k_scales[pb * Hkv + kvh]);
            vs = v_scales[pb * Hkv + kvh];
        }
        const float m_new = fmaxf(m, wave_max(s));
        const float m_safe = m_new == -INFINITY ? 0.0f : m_new;  // keys that all score -inf weigh nothing
        const float alpha = expf(m - m_safe);
        const float p = key < keys ? expf(s - m_safe) : 0.0f;
        float ps = p;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) ps += __shfl_xor(ps, x);
        l = l * alpha + ps;
        m = m_new;
        p_s[wave][lane] = p * vs;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= alpha;
        const int n = (int)(keys - base < 64 ? keys - base : 64);
        if (wide) {
            if (vr < together)
                for (int j = vr; j < n; j += together) {
                    float x[4];
                    decode4<F>(*reinterpret_cast<const unsigned *>(v_cache + row_s[wave][j] + 4 * vc), x);
                    const float pw = p_s[wave][j];
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] += pw * x[i];
                }
        } else {
            for (int j = 0; j < n; ++j) {
                const float pw = p_s[wave][j];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (vc + 64 * i < D) o[i] += pw * decode1<F>(v_cache[row_s[wave][j] + vc + 64 * i]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    // join: the lanes of a wave that hold the same dims, then the waves
    if (lane == 0) {
        m_s[wave] = m;
        l_s[wave] = l;
    }
    for (int r = 0; r < together; ++r) {
        if (vr == r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = wide ? 4 * vc + i : vc + 64 * i;
                if (d < D) o_s[wave][d] += o[i];
            }
        __syncthreads();
    }
    const float mx = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
    float L = 0.0f, y = 0.0f;
    const int d = threadIdx.x;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = m_s[w] == -INFINITY ? 0.0f : expf(m_s[w] - mx);
        L += f * l_s[w];
        y += f * o_s[w][d];
    }
    if (d < D) out[orow + d] = static_cast<ET>(L > 0.0f ? y / L : 0.0f);
}

template <typename ET, Kv8Format F>
hipError_t launch_generic(const PagedAttnArgs &a, const float *ks, const float *vs, hipStream_t stream) {
    const int64_t rows = (int64_t)a.num_heads * a.num_new_tokens;
    if (rows > 0x7fffffffLL) return hipErrorInvalidValue;
    const auto at4 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; };
    const bool wide = a.head_dim % 4 == 0 && at4(a.k_cache) && at4(a.v_cache);
    paged_attn_kv8_generic_kernel<ET, F><<<dim3((unsigned)rows, a.num_seqs), dim3(256), 0, stream>>>(
        static_cast<const ET *>(a.q), static_cast<const unsigned char *>(a.k_cache),
        static_cast<const unsigned char *>(a.v_cache), ks, vs, a.block_tables, a.context_lens,
        static_cast<ET *>(a.out), a.num_new_tokens, a.num_heads, a.num_kv_heads, a.head_dim, a.block_size,
        a.max_blocks_per_seq, a.num_cache_blocks, a.scale, wide);
    return hipGetLastError();
}

}  // namespace

PagedKv8Path paged_attn_kv8_path(DType, const PagedAttnArgs &) { return PagedKv8Path::Generic; }

size_t paged_attn_kv8_workspace_bytes(DType, const PagedAttnArgs &) { return 0; }

hipError_t launch_paged_attn_kv8(DType dt, Kv8Format fmt, const PagedAttnArgs &a, const float *k_scales,
                                 const float *v_scales, hipStream_t stream) {
    if (a.num_seqs <= 0) return hipSuccess;
    if (dt == DType::BF16)
        return fmt == Kv8Format::Int8 ? launch_generic<__bf16, Kv8Format::Int8>(a, k_scales, v_scales, stream)
                                      : launch_generic<__bf16, Kv8Format::E4M3>(a, k_scales, v_scales, stream);
    return fmt == Kv8Format::Int8 ? launch_generic<float, Kv8Format::Int8>(a, k_scales, v_scales, stream)
                                  : launch_generic<float, Kv8Format::E4M3>(a, k_scales, v_scales, stream);
}

}  // namespace kernels
}  // namespace nvllm

// paged_attn_kv8.hip -- paged attention over the 8-bit KV cache (gfx950).
//
// The block tables, context lengths and the bottom-right causal mask are those of paged_attn.hip
// (reference src/attention/paged.rs:117-192, :357-381); K and V are codes with one scale per (block,
// kv head), kv8_common.hpp:
//   s_ij = softmax_scale * kscale[block of j] * (q_i . kcode_j),   p_ij = exp(s_ij - max_j s_ij)
//   o_i  = sum_j (p_ij * vscale[block of j]) vcode_j / sum_j p_ij
// A scale belongs to a token (its block), so K's multiplies scores.  What the matrix unit gets of K is the
// code in its type, exactly; of V the code times the power of two in its scale, exactly too.
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
// token, query head); its W waves take every W-th tile of 64 keys and join at the end.  f32 FMA.
// A lane is a key for q.k and four dims for p.v.  `vec`: bytes of K a load takes (16, 4, 1; V at most 4).
// Bound by latency, and by the arithmetic where there is work for the whole chip (K and V are read and converted
// once per query head): the table's entry is read a tile ahead and eight rows of V are on their way during q.k
// (64 x 1024, head_dim 128, f32: 98 -> 61 us).
// ---------------------------------------------------------------------------
// block id as the kernels use it: inside the pool
__device__ __forceinline__ int pool_id(int id, int64_t num_cache_blocks) {
    const int most = (int)num_cache_blocks - 1;  // the C entries refuse larger pools
    return id < 0 ? 0 : (id > most ? most : id);
}

// A tile with a V scale of 2^64 or more takes its exponents from a reference at least kLift (a power of two) above the
// row's maximum, so that there p <= 2^-32.  Then nothing overflows, whatever the finite scales: values are below 2^128 and
// a walk has 2^30 keys at most, so these tiles' sums stay below 2^(30 - 32 + 128), and the others', whose p may be 2^14
// (kSlack below) and whose codes are below 2^9, below 2^(30 + 14 + 64 + 9).  The output is divided by the sum of
// the same p, so their size cancels; lost is what is below 2^-94, p of the largest p or p * scale.
constexpr float kLift = 32.0f;
constexpr float kLarge = 0x1p64f;

constexpr int kAtOnce = 8;  // rows of V that a group of lanes has on their way

// what lanes of the wave wrote to LDS before, lanes of it may read after
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename ET, Kv8Format F, int W>
__global__ __launch_bounds__(64 * W) void paged_attn_kv8_generic_kernel(
    const ET *__restrict__ q, const unsigned char *__restrict__ k_cache, const unsigned char *__restrict__ v_cache,
    const float *__restrict__ k_scales, const float *__restrict__ v_scales, const int32_t *__restrict__ block_tables,
    const int32_t *__restrict__ context_lens, ET *__restrict__ out, int T, int Hq, int Hkv, int D, int block_size,
    int max_blocks_per_seq, int64_t num_cache_blocks, float scale, int vec) {
    __shared__ float q_s[256];
    __shared__ float p_s[W][64];
    __shared__ int64_t row_s[W][64];  // element offset of each key's row
    __shared__ float o_s[W][256];
    __shared__ float m_s[W], l_s[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = (int)(blockIdx.x % (unsigned)Hq), t = (int)(blockIdx.x / (unsigned)Hq), seq = blockIdx.y;
    const int kvh = h / (Hq / Hkv);
    int ctx = context_lens[seq];
    const int64_t cap = (int64_t)max_blocks_per_seq * block_size;
    if (ctx > cap) ctx = (int)cap;  // never read past the table row
    if (ctx < 0) ctx = 0;
    const int keys = ctx - T + t + 1;  // keys this query sees: 0 .. keys - 1 (none if <= 0)
    const int64_t orow = (((int64_t)seq * T + t) * Hq + h) * D;
    const bool wide = vec >= 4;
    if (threadIdx.x < 256) q_s[threadIdx.x] = (int)threadIdx.x < D ? to_f32(q[orow + threadIdx.x]) : 0.0f;
    for (int d = lane; d < 256; d += 64) o_s[wave][d] = 0.0f;
    __syncthreads();
    const int32_t *table = block_tables + (int64_t)seq * max_blocks_per_seq;
    const int lanes = wide ? D / 4 : 64, together = wide ? 64 / lanes : 1;  // lanes per V row, rows at once
    const int vr = wide ? lane / lanes : 0, vc = wide ? lane % lanes : lane;
    float m = -INFINITY, l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    int base = 64 * wave;
    int64_t pb = base + lane < keys ? pool_id(table[(base + lane) / block_size], num_cache_blocks) : 0;
    for (; base < keys; base += 64 * W) {
        const int key = base + lane, n = keys - base < 64 ? keys - base : 64;
        // a lane without a key takes the tile's first (its weight is 0)
        const int64_t at = ((pb * block_size + key % block_size) * Hkv + kvh) * D;
        const int64_t first = __shfl(at, 0), row = key < keys ? at : first;
        row_s[wave][lane] = row;
        const float ks = key < keys ? k_scales[pb * Hkv + kvh] : 0.0f, vs = key < keys ? v_scales[pb * Hkv + kvh] : 0.0f;
        const int next = key + 64 * W;
        pb = next < keys ? pool_id(table[next / block_size], num_cache_blocks) : 0;
        wave_sync();
        unsigned v[kAtOnce];  // on their way during q.k and the softmax
        const auto load_v = [&](int j0) {
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const int r = j0 + j * together + vr;
                v[j] = *reinterpret_cast<const unsigned *>(v_cache + row_s[wave][r < 64 ? r : 0] + 4 * vc);
            }
        };
        if (wide) load_v(0);
        float acc = 0.0f;
        if (vec == 16) {
#pragma unroll 4
            for (int d = 0; d < D; d += 16) {
                const u32x4 w = *reinterpret_cast<const u32x4 *>(k_cache + row + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x[4];
                    decode4<F>(w[e], x);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc += q_s[d + 4 * e + i] * x[i];
                }
            }
        } else if (wide) {
            for (int d = 0; d < D; d += 4) {
                float x[4];
                decode4<F>(*reinterpret_cast<const unsigned *>(k_cache + row + d), x);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc += q_s[d + i] * x[i];
            }
        } else {
            for (int d = 0; d < D; ++d) acc += q_s[d] * decode1<F>(k_cache[row + d]);
        }
        const float s = key < keys ? acc * (scale * ks) : -INFINITY;
        const float m_new = fmaxf(m, wave_max(s) + (__any(vs >= kLarge) ? kLift * 0.6931472f : 0.0f));
        const float m_safe = m_new == -INFINITY ? 0.0f : m_new;  // keys that all score -inf weigh nothing
        const float alpha = expf(m - m_safe);
        const float p = key < keys ? expf(s - m_safe) : 0.0f;
        l = l * alpha + p;  // the lane's own keys; joined at the end
        m = m_new;
        p_s[wave][lane] = p * vs;
        wave_sync();
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= alpha;
        if (wide) {
            for (int j0 = 0; j0 < n; j0 += kAtOnce * together) {
                if (j0 > 0) load_v(j0);
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const int r = j0 + j * together + vr;
                    if (vr >= together || r >= n) continue;
                    float x[4];
                    decode4<F>(v[j], x);
                    const float pw = p_s[wave][r];
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] += pw * x[i];
                }
            }
        } else {
            for (int j = 0; j < n; ++j) {
                const float pw = p_s[wave][j];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (vc + 64 * i < D) o[i] += pw * decode1<F>(v_cache[row_s[wave][j] + vc + 64 * i]);
            }
        }
        wave_sync();
    }
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x);
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
        wave_sync();
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    float mx = m_s[0], L = 0.0f, y = 0.0f;
#pragma unroll
    for (int w = 1; w < W; ++w) mx = fmaxf(mx, m_s[w]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float f = m_s[w] == -INFINITY ? 0.0f : expf(m_s[w] - mx);
        L += f * l_s[w];
        y += f * o_s[w][d];
    }
    out[orow + d] = static_cast<ET>(L == 0.0f ? 0.0f : y / L);  // no key seen: zeros
}

// Sixteen waves where a workgroup has a CU to itself and long tables (int8, f32, head_dim 64, 8 heads, us with 4 and 16
// waves: 9 x 777 T = 3 14.9 and 10.1, 1 x 4000 47 and 22, 1 x 500 9.7 and 8.5, 1 x 250 6.9 and 7.7; 64 x 1024 with 16
// heads 49 and 59).
int generic_waves(const PagedAttnArgs &a) {
    const int64_t groups = (int64_t)a.num_seqs * a.num_new_tokens * a.num_heads;
    return groups <= device_cus() && (int64_t)a.max_blocks_per_seq * a.block_size > 512 ? 16 : 4;
}

template <typename ET, Kv8Format F>
hipError_t launch_generic(const PagedAttnArgs &a, const float *ks, const float *vs, hipStream_t stream) {
    const int64_t rows = (int64_t)a.num_heads * a.num_new_tokens;
    if (rows > 0x7fffffffLL) return hipErrorInvalidValue;
    const auto aligned = [&](unsigned n) {
        return a.head_dim % n == 0 && ((reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) & (n - 1)) == 0;
    };
    const int vec = aligned(16) ? 16 : aligned(4) ? 4 : 1;
#define NVLLM_KV8_GENERIC(W)                                                                                        \
    paged_attn_kv8_generic_kernel<ET, F, W><<<dim3((unsigned)rows, a.num_seqs), dim3(64 * W), 0, stream>>>(         \
        static_cast<const ET *>(a.q), static_cast<const unsigned char *>(a.k_cache),                                \
        static_cast<const unsigned char *>(a.v_cache), ks, vs, a.block_tables, a.context_lens,                      \
        static_cast<ET *>(a.out), a.num_new_tokens, a.num_heads, a.num_kv_heads, a.head_dim, a.block_size,          \
        a.max_blocks_per_seq, a.num_cache_blocks, a.scale, vec)
    if (generic_waves(a) == 16) NVLLM_KV8_GENERIC(16);
    else NVLLM_KV8_GENERIC(4);
#undef NVLLM_KV8_GENERIC
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Decode path: bf16, head_dim 128, block_size 16, up to 48 query rows (T * Hq/Hkv) per kv head.
//
// Bound by HBM: a cached token costs 2 * Hkv * 128 bytes, half of the bf16 cache's.  A workgroup has one kv head
// of one sequence, its W waves a part of the keys each (all query rows of the head), and they join through LDS at
// the end: one launch, no workspace.  Only where (sequence, kv head) pairs are few or walks long are the keys split
// over workgroups as well, with partials and a merge launch as in paged_attn.hip.  (Waves for the heads of a sequence
// instead, which read whole blocks together, as the bf16 kernel has them: 256 x 2048 int8 184 against 166 us,
// 64 x 4096 with 4 splits 91 against 95; short walks even out better.)  What one byte a value changes:
//   tile    32 keys (2 blocks), 8 KiB.  One in registers, the next on its way (two or three ahead: 256 x 2048 the
//           same, 256 x 512 T = 12 92 against 84 us, 16 x 2048 17.8 against 16.3);
//   K       8 lanes x 16 B read a 128-byte row, 8 rows an instruction; through the wave's LDS image (16-byte
//           chunk ch of row r at position ch ^ (r & 7): 8 rows x 1 chunk and 1 row x 8 chunks both touch
//           all banks once).  A lane reads chunks 4i + g of row c: 16 dims = two MFMA k-steps of 8, so the
//           dims are in an order of their own and Q's fragments follow it;
//   V       the same image; ds_read_b64_tr_b8 gives a lane 8 keys of one dim.  Group g takes the keys that
//           its scores are for (4g .. 4g+3 of two blocks), so P needs no lane movement;
//   codes   become bf16 (K) and f16 (V) in registers, exactly (v_cvt_scalef32_pk_bf16_fp8 and _f16_fp8, two a
//           instruction; int8 by way of f32, or of f16's bits), and go to mfma_f32_16x16x32;
//   scales  lane l of the wave holds id, K scale and V scale of block l of a run of 64; v_readlane makes
//           them scalars at the tile that needs them.  The next run's are loaded 32 tiles ahead.
// ---------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) int i32x2;

constexpr int kD = 128;
constexpr int kBS = 16;
constexpr int kTileBlocks = 2;
constexpr int kTileKeys = kTileBlocks * kBS;
constexpr int kImage = kTileKeys * kD;  // 4 KiB: one tile of K or of V
constexpr int kRun = 64;                // blocks whose ids and scales a wave holds at once
constexpr int kMaxDecodeRows = 48;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// lane l's value and lane l ^ 32's.  In asm: given the builtin the same value twice, hipcc takes its two
// results for equal.  s_nop 1 = the wait states between a vector write and the swap; the swap itself needs
// none before its results are read.
__device__ __forceinline__ void swap_halves(float &a, float &b) {
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
// the same for lanes l and l ^ 16
__device__ __forceinline__ void swap_rows(float &a, float &b) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ float half_max(float x) {
    float a = x, b = x;
    swap_halves(a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float half_sum(float x) {
    float a = x, b = x;
    swap_halves(a, b);
    return a + b;
}

// over the four lanes l ^ {0, 16, 32, 48}
__device__ __forceinline__ float quad_max(float x) {
    float a = x, b = x;
    swap_rows(a, b);
    return half_max(fmaxf(a, b));
}

// Weights and values go to the matrix unit in f16.  The codes of both formats times a power of two from 2^-15 to 2^5 are
// f16 numbers, so V is exact, and a weight is off by 2^-11 of itself.  f16 has little range; p therefore uses it to
// its end: exponents are taken from a reference that is moved to kRoom below a row's maximum, and only when that has
// passed it by kSlack, so that the largest p is 2^7 .. 2^14, most tiles rescale nothing, and a p that f16 does not hold
// in full is off by 2^-32 of the largest.  (In bf16, which needs none of this, a weight is off by 2^-8 and the
// output's error against 64 bits a third larger: 2.3e-3 for 1.7e-3.)
// A V scale that is no power of two (no write makes one): the decode kernel multiplies p by its fraction, 1 .. 2 (to 2^15).
// A tile with a scale out of the range ("wild"; to the tile kernel one that is no power of two, too) takes bf16 instead, p
// times scale and the bare code; so does every tile after one that lifted the reference, where p is small.
constexpr float kSlack = 14.0f, kRoom = 7.0f;

// whether a block of this V scale goes through f16
template <bool POWERS> __device__ __forceinline__ bool tame(float scale) {
    const unsigned b = __builtin_bit_cast(unsigned, scale), lo = 0x38000000u, hi = 0x42800000u;  // 2^-15, 2^6
    return b == 0 || (b - lo < hi - lo && (!POWERS || (b & 0x7fffffu) == 0));
}
// scale = power * fraction, 1 <= fraction < 2 (a scale of 0: power 0)
__device__ __forceinline__ float power_of(float scale) {
    return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, scale) & 0xff800000u);
}
__device__ __forceinline__ float fraction_of(float scale) {
    return __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, scale) & 0x7fffffu) | 0x3f800000u);
}

// A kv head's rows of a cache block as a buffer: 16 bytes of it at lane_offset + row_offset, zeros without a
// memory access if `valid` is false.  Tiles past the end are "loaded" that way, so that every step of a loop
// issues the same loads: behind a load that a branch may skip, hipcc's waits count only what is outstanding on
// the branch that skipped it, and so wait for the newest tile as well.  (It also keeps addresses scalar.)
typedef __amdgpu_buffer_rsrc_t Rows;
__device__ __forceinline__ Rows block_rows(const unsigned char *base, int64_t offset, int bytes, bool valid) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(base + offset), 0, valid ? bytes : 0, 0x00027000);
}
template <bool STREAM> __device__ __forceinline__ u32x4 load16(Rows rows, unsigned lane_offset, unsigned row_offset) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, lane_offset, row_offset, STREAM ? 2 : 0));
}

// A wave's view of its part of a block table: lane l holds id and scales of block `base + l` of a run of 64, and
// the next run's are on their way.  What is loaded is looked at (clamped, masked) only when its run begins, so
// that nothing waits for it before.  Past the part's end: the last id (read, and masked), scale 0.
template <bool POWERS> struct Run {
    const int32_t *table;
    const float *k_scales, *v_scales;  // of the kv head: + Hkv * id
    int Hkv, end, lane;
    int64_t num_cache_blocks;
    int id, id_n, id_nn;               // id_nn: as the table has it
    float ks, vs, ks_n, vs_n;          // _n: as loaded
    unsigned long long wild, large;    // bit l: V scale of block base + l is not tame / is kLarge or more

    __device__ __forceinline__ int raw_id(int base) const {
        const int j = base + lane;
        return table[j < end ? j : end - 1];
    }
    __device__ __forceinline__ void ask_scales(int ids, float &a, float &b) const {
        a = k_scales[(int64_t)ids * Hkv];
        b = v_scales[(int64_t)ids * Hkv];
    }
    __device__ __forceinline__ void begin(int base) {
        id = pool_id(raw_id(base), num_cache_blocks);
        id_n = pool_id(raw_id(base + kRun), num_cache_blocks);
        id_nn = raw_id(base + 2 * kRun);
        ask_scales(id, ks, vs);
        if (base + lane >= end) ks = vs = 0.0f;
        look();
        ask_scales(id_n, ks_n, vs_n);
    }
    __device__ __forceinline__ void look() {
        wild = __ballot(!tame<POWERS>(vs));
        large = __ballot(vs >= kLarge);
    }
    __device__ __forceinline__ void advance(int base) {  // base: the run that begins
        id = id_n;
        ks = base + lane < end ? ks_n : 0.0f;
        vs = base + lane < end ? vs_n : 0.0f;
        look();
        id_n = pool_id(id_nn, num_cache_blocks);
        ask_scales(id_n, ks_n, vs_n);
        id_nn = raw_id(base + 2 * kRun);
    }
    __device__ __forceinline__ int64_t id_at(int j) const { return __builtin_amdgcn_readlane(id, j); }
    __device__ __forceinline__ float k_at(int j) const {
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ks), j));
    }
    __device__ __forceinline__ float v_at(int j) const {
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, vs), j));
    }
};

// 8 codes -> 8 bf16, exact
template <Kv8Format F> __device__ __forceinline__ bf16x8 widen8(unsigned w0, unsigned w1) {
    u32x4 r;
    if constexpr (F == Kv8Format::E4M3) {
        r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, false));
        r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, true));
        r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, false));
        r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, true));
    } else {
        float x[8];
        decode4<F>(w0, x);
        decode4<F>(w1, x + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    }
    return __builtin_bit_cast(bf16x8, r);
}

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

// a tame block's codes times its scale, exact; `two`: the scale twice, in f16
__device__ __forceinline__ f16x2 twice(float scale) { return f16x2{(_Float16)scale, (_Float16)scale}; }
template <Kv8Format F> __device__ __forceinline__ void scaled4(unsigned w, float scale, f16x2 two, f16x2 &a, f16x2 &b) {
    if constexpr (F == Kv8Format::E4M3) {
        a = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
        b = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true));
    } else {
        // 0x6400 + u is 1024 + u; u = code + 128
        const f16x2 off = two * (_Float16)-1152.0f;
        const unsigned u = w ^ 0x80808080u;
        a = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)), two, off);
        b = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)), two, off);
    }
}
template <Kv8Format F> __device__ __forceinline__ f16x8 scaled8(unsigned w0, unsigned w1, const float (&scale)[2], const f16x2 (&two)[2]) {
    f16x2 x[4];
    scaled4<F>(w0, scale[0], two[0], x[0], x[1]);
    scaled4<F>(w1, scale[1], two[1], x[2], x[3]);
    return __builtin_bit_cast(f16x8, x);
}

// weights as the matrix unit takes them, in either type
__device__ __forceinline__ u32x4 halves(const float (&p)[8]) {
    f16x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (_Float16)p[i];
    return __builtin_bit_cast(u32x4, r);
}
__device__ __forceinline__ u32x4 bfloats(const float (&p)[8]) {
    return u32x4{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])};
}

// hipcc leaves too few wait states between the last matrix instruction of a basic block and a read of
// its result in the next one (seen here as wrong values of one accumulator register; tests/mfma_waits.py
// finds such places in the assembly).  Behind code whose results leave a block: 8 wait states.
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 7");
    __builtin_amdgcn_sched_barrier(0);
}

struct Tile {
    u32x4 k[kTileBlocks][2], v[kTileBlocks][2];  // [block][rows 0-7, 8-15]
    float ks[kTileBlocks], vs[kTileBlocks];      // wave-uniform
    bool wild, large;                            // and so are these: goes through bf16; lifts the reference
};

// byte c of the result is 0xff where byte c of w is an E4M3 NaN (0x7f, 0xff)
__device__ __forceinline__ unsigned nan_bytes(unsigned w) {
    const unsigned t = (w & 0x7f7f7f7fu) + 0x01010101u;  // bit 7 of a byte: its low seven bits were all ones
    return ((t & 0x80808080u) >> 7) * 0xffu;
}

// NQT query tiles of 16 rows.  One and two leave room for two waves a SIMD and more (two in workgroups of four waves
// against one wave a SIMD in workgroups of two: 256 x 2048 T = 8 213 -> 194 us, 128 x 512 38 -> 32, 4 x 4096 19 -> 15;
// 64 x 4096 99 -> 104); three need a SIMD's registers.
template <Kv8Format F, int NQT, int W, bool STREAM>
__global__ __launch_bounds__(64 * W, NQT <= 2 ? 2 : 1) void paged_attn_kv8_decode_kernel(
    const __bf16 *__restrict__ q, const unsigned char *__restrict__ k_cache, const unsigned char *__restrict__ v_cache,
    const float *__restrict__ k_scales, const float *__restrict__ v_scales, const int32_t *__restrict__ block_tables,
    const int32_t *__restrict__ context_lens, __bf16 *__restrict__ out, float *__restrict__ ws_o,
    float *__restrict__ ws_ml, int T, int Hq, int Hkv, int max_blocks_per_seq, int64_t num_cache_blocks,
    float scale, int num_splits, int blocks_per_split) {
    __shared__ __attribute__((aligned(16))) unsigned char lds_all[W * NQT * 8192];  // images; parts to join
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c = lane & 15;
    const int split = blockIdx.x, seq = blockIdx.y;
    const int kvh = blockIdx.z;

    const int G = Hq / Hkv, R = T * G;
    int ctx = context_lens[seq];
    const int64_t cap = (int64_t)max_blocks_per_seq * kBS;
    if (ctx > cap) ctx = (int)cap;  // never read past the table row
    if (ctx < 0) ctx = 0;
    const int nblk_seq = ctx > 0 ? (int)(((int64_t)ctx + kBS - 1) / kBS) : 0;
    int blk_begin = split * blocks_per_split;
    int blk_end = blk_begin + blocks_per_split;
    if (blk_end > nblk_seq) blk_end = nblk_seq;
    // this wave's part, in whole tiles
    const int all = blk_end > blk_begin ? blk_end - blk_begin : 0;
    const int part = ((all + W - 1) / W + kTileBlocks - 1) / kTileBlocks * kTileBlocks;
    blk_begin += wave * part;
    if (blk_end > blk_begin + part) blk_end = blk_begin + part;
    const int ntiles = blk_end > blk_begin ? (blk_end - blk_begin + kTileBlocks - 1) / kTileBlocks : 0;
    unsigned char *lds_k = lds_all + wave * 2 * kImage, *lds_v = lds_k + kImage;
    const int32_t *table = block_tables + (int64_t)seq * max_blocks_per_seq;

    // Q^T fragments (B operand): k-step 2i + h of lane (g, c) holds Q[row c][16 (4i + g) + 8h .. + 7]
    bf16x8 qf[NQT][4];
    int t_of_row[NQT];
    const unsigned flip = scale < 0.0f ? 0x80008000u : 0u;  // a negative scale moves into Q: factors stay >= 0
    const float scale_log2e = fabsf(scale) * 1.4426950408889634f;
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        const int r = qt * 16 + c;
        const int t = r < R ? r / G : 0, hg = r < R ? r - t * G : 0;
        t_of_row[qt] = t;
        const __bf16 *qrow = q + (((int64_t)seq * T + t) * Hq + kvh * G + hg) * kD;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            u32x4 x = {0u, 0u, 0u, 0u};
            if (r < R) x = *reinterpret_cast<const u32x4 *>(qrow + 16 * (4 * (s >> 1) + g) + 8 * (s & 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] ^= flip;
            qf[qt][s] = __builtin_bit_cast(bf16x8, x);
        }
    }

    const int64_t block_bytes = (int64_t)kBS * Hkv * kD;
    const unsigned row_stride = (unsigned)Hkv * kD;
    const int lr = lane >> 3, lch = lane & 7;
    const int head_bytes = (kBS - 1) * (int)row_stride + kD;  // from a head's first byte of a block to its last
    const unsigned lane_off = (unsigned)lr * row_stride + 16u * lch;
    const unsigned wr = (unsigned)(lr * kD + 16 * (lch ^ lr));                    // + 2048 b + 1024 i
    const unsigned krd0 = (unsigned)(c * kD + 16 * (g ^ (c & 7)));                // + 2048 b, chunk g
    const unsigned krd1 = (unsigned)(c * kD + 16 * ((4 + g) ^ (c & 7)));          // chunk 4 + g
    const int tr_q = c >> 1;                                                      // transposed read: its row
    const int tr_row = (tr_q < 4 ? 0 : kBS) + 4 * g + (tr_q & 3);
    const unsigned tr_base = (unsigned)(tr_row * kD + 8 * (c & 1));
    const unsigned tr_sw = (unsigned)(tr_row & 7);

    Run<false> run{table, k_scales + kvh, v_scales + kvh, Hkv, blk_end, lane, num_cache_blocks};
    bool lifted = false;
    auto load_tile = [&](Tile &tl, int t) {
        const int j = (kTileBlocks * t) & (kRun - 1);
        tl.large = (run.large >> j & ((1u << kTileBlocks) - 1)) != 0;
        lifted |= tl.large;
        tl.wild = (run.wild >> j & ((1u << kTileBlocks) - 1)) != 0 || lifted;
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b) {
            tl.ks[b] = run.k_at(j + b);
            tl.vs[b] = run.v_at(j + b);
            const int64_t at = run.id_at(j + b) * block_bytes + kvh * kD;
            const Rows k = block_rows(k_cache, at, head_bytes, t < ntiles), v = block_rows(v_cache, at, head_bytes, t < ntiles);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                tl.k[b][i] = load16<STREAM>(k, lane_off, 8 * i * row_stride);
                tl.v[b][i] = load16<STREAM>(v, lane_off, 8 * i * row_stride);
            }
        }
        if (j == kRun - kTileBlocks) run.advance(blk_begin + kTileBlocks * (t + 1));
    };

    float m_run[NQT], l_run[NQT];
    f32x4 acc[NQT][8];
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        m_run[qt] = -INFINITY;
        l_run[qt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) acc[qt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int first_masked = ctx - (T - 1);  // first key that some query row cannot see
    unsigned nan_seen = 0;                   // among the values of the tiles from there on

    // A operand of P.V, as codes: 8 keys (4g .. 4g+3 of both blocks) of dim 16 dt + c
    auto v_codes = [&](int dt) -> i32x2 {
        typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
        return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)(lds_v + tr_base + 16u * ((unsigned)dt ^ tr_sw)));
    };
    auto v_fragment = [&](int dt) -> bf16x8 {
        const i32x2 w = v_codes(dt);
        return widen8<F>((unsigned)w[0], (unsigned)w[1]);
    };
    auto compute_tile = [&](Tile &tl, int t) {
        const int blk0 = blk_begin + kTileBlocks * t, key0 = blk0 * kBS;
        const bool tail = key0 + kTileKeys > first_masked || blk0 + kTileBlocks > blk_end;
        if (tail) {  // V rows past the context hold anything: zeros, so that 0 * them is 0
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (key0 + b * kBS + 8 * i + lr >= ctx || blk0 + b >= blk_end) tl.v[b][i] = u32x4{0u, 0u, 0u, 0u};
                    if constexpr (F == Kv8Format::E4M3)  // and so for a NaN that only some rows see (below)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const unsigned n = nan_bytes(tl.v[b][i][w]);
                            nan_seen |= n;
                            tl.v[b][i][w] &= ~n;
                        }
                }
        }
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4 *>(lds_k + wr + 2048 * b + 1024 * i) = tl.k[b][i];
        // S^T = K Q^T, one 16 x 16 tile per block
        f32x4 s[NQT][kTileBlocks];
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b) {
            const u32x4 k0 = *reinterpret_cast<const u32x4 *>(lds_k + krd0 + 2048 * b);
            const u32x4 k1 = *reinterpret_cast<const u32x4 *>(lds_k + krd1 + 2048 * b);
            const bf16x8 a0 = widen8<F>(k0[0], k0[1]), a1 = widen8<F>(k0[2], k0[3]);
            const bf16x8 a2 = widen8<F>(k1[0], k1[1]), a3 = widen8<F>(k1[2], k1[3]);
#pragma unroll
            for (int qt = 0; qt < NQT; ++qt) {
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
                x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, qf[qt][0], x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, qf[qt][1], x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a2, qf[qt][2], x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a3, qf[qt][3], x, 0, 0, 0);
                s[qt][b] = x;
            }
        }
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i) *reinterpret_cast<u32x4 *>(lds_v + wr + 2048 * b + 1024 * i) = tl.v[b][i];
        // online softmax in the exp2 domain; a query row's state lives in the lanes c = row
        float f[kTileBlocks];
#pragma unroll
        for (int b = 0; b < kTileBlocks; ++b) f[b] = tl.ks[b] * scale_log2e;
        if (tail) {
#pragma unroll
            for (int qt = 0; qt < NQT; ++qt)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool see = key0 + (j >> 2) * kBS + 4 * g + (j & 3) <= ctx - T + t_of_row[qt] &&
                                     blk0 + (j >> 2) < blk_end;
                    s[qt][j >> 2][j & 3] = see ? s[qt][j >> 2][j & 3] * f[j >> 2] : -INFINITY;
                }
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b) f[b] = 1.0f;
        }
        const float slack = tl.large ? -kLift : kSlack, above = tl.large ? kLift : -kRoom;
#pragma unroll
        for (int qt = 0; qt < NQT; ++qt) {
            float mx = -INFINITY;
#pragma unroll
            for (int b = 0; b < kTileBlocks; ++b)  // factors are >= 0
                mx = fmaxf(mx, f[b] * fmaxf(fmaxf(s[qt][b][0], s[qt][b][1]), fmaxf(s[qt][b][2], s[qt][b][3])));
            mx = quad_max(mx);
            if (__any(mx > m_run[qt] + slack)) {
                const float m_new = fmaxf(m_run[qt], mx + above);
                const float alpha = m_new == -INFINITY ? 1.0f : fast_exp2(m_run[qt] - m_new);
                m_run[qt] = m_new;
                l_run[qt] *= alpha;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) acc[qt][dt] *= alpha;
            }
        }
        // weights of a query tile (their sum goes into l_run)
        const auto weights = [&](int qt, float (&p)[8]) {
            const float m_safe = m_run[qt] == -INFINITY ? 0.0f : m_run[qt];
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[j] = fast_exp2(fmaf(s[qt][j >> 2][j & 3], f[j >> 2], -m_safe));
                sum += p[j];
            }
            l_run[qt] += sum;
        };
        float vs[kTileBlocks] = {tl.vs[0], tl.vs[1]};
        if (__builtin_expect(tl.wild, 0)) {  // (here, so that no branch is between the weights and the f16 product: T = 12 281 -> 261 us)
#pragma unroll
            for (int qt = 0; qt < NQT; ++qt) {
                float p[8];
                weights(qt, p);
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] *= vs[j >> 2];
                const bf16x8 pw = __builtin_bit_cast(bf16x8, bfloats(p));
#pragma unroll
                for (int dt = 0; dt < 8; ++dt)
                    acc[qt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v_fragment(dt), pw, acc[qt][dt], 0, 0, 0);
                // nothing is left for the rest of the tile's work
#pragma unroll
                for (int j = 0; j < 8; ++j) s[qt][j >> 2][j & 3] = -INFINITY;
            }
            f[0] = f[1] = vs[0] = vs[1] = 1.0f;
            settle();
        }
        u32x4 pf[NQT];
        const float fraction[kTileBlocks] = {fraction_of(vs[0]), fraction_of(vs[1])};
#pragma unroll
        for (int qt = 0; qt < NQT; ++qt) {
            float p[8];
            weights(qt, p);
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] *= fraction[j >> 2];
            pf[qt] = halves(p);
        }
        // O^T += V^T P^T
        vs[0] = power_of(vs[0]);
        vs[1] = power_of(vs[1]);
        const f16x2 two[2] = {twice(vs[0]), twice(vs[1])};
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            const i32x2 w = v_codes(dt);
            const f16x8 a = scaled8<F>((unsigned)w[0], (unsigned)w[1], vs, two);
#pragma unroll
            for (int qt = 0; qt < NQT; ++qt)
                acc[qt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, __builtin_bit_cast(f16x8, pf[qt]), acc[qt][dt], 0, 0, 0);
        }
        settle();
    };

    if (ntiles > 0) {
        run.begin(blk_begin);
        Tile tl[2];
        load_tile(tl[0], 0);
        for (int t = 0; t < ntiles; t += 2)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                load_tile(tl[1 - u], t + u + 1);
                if (t + u < ntiles) compute_tile(tl[u], t + u);
            }
    }

    if constexpr (F == Kv8Format::E4M3)
        if (__any(nan_seen != 0)) {
            // A NaN among values that some rows must not see (0 * NaN would have reached them, so the loop took it for
            // 0): which (dim, row) pairs do see one is a product of zeros and ones.
            for (int t = 0; t < ntiles; ++t) {
                const int blk0 = blk_begin + kTileBlocks * t, key0 = blk0 * kBS;
                if (key0 + kTileKeys <= first_masked && blk0 + kTileBlocks <= blk_end) continue;
#pragma unroll
                for (int b = 0; b < kTileBlocks; ++b)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        u32x4 one = {0u, 0u, 0u, 0u};
                        if (key0 + b * kBS + 8 * i + lr < ctx && blk0 + b < blk_end) {
                            const int64_t at = pool_id(table[blk0 + b], num_cache_blocks) * block_bytes + kvh * kD;
                            one = *reinterpret_cast<const u32x4 *>(v_cache + at + 8 * i * row_stride + lane_off);
#pragma unroll
                            for (int w = 0; w < 4; ++w) one[w] = nan_bytes(one[w]) & 0x38383838u;  // 1.0
                        }
                        *reinterpret_cast<u32x4 *>(lds_v + wr + 2048 * b + 1024 * i) = one;
                    }
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) {
                    const bf16x8 one = v_fragment(dt);
#pragma unroll
                    for (int qt = 0; qt < NQT; ++qt) {
                        u32x4 see;
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const int key = key0 + (e >> 2) * kBS + 4 * g + (e & 3), last = ctx - T + t_of_row[qt];
                            see[e >> 1] = (key <= last ? 0x3f80u : 0u) | (key + 1 <= last ? 0x3f800000u : 0u);
                        }
                        const f32x4 hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(one, __builtin_bit_cast(bf16x8, see),
                                                                                  f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[qt][dt][e] = hit[e] > 0.0f ? __builtin_nanf("") : acc[qt][dt][e];
                    }
                }
                settle();
            }
        }

    // join the waves' parts: wave w sums the dims [128 / W w, ..) of all of them, so every wave leaves the others' dims
    // (and each row's m and l) in LDS, a lane's 16 bytes where the same lane of the reader finds them
    __shared__ float ml[W][NQT * 16][2];
    constexpr int kOwn = 8 / W;  // dt a wave sums
    const auto part_of = [&](int w, int qt, int dt) {
        return reinterpret_cast<f32x4 *>(lds_all + ((w * NQT + qt) * 8 + dt) * 1024 + 16 * lane);
    };
    __syncthreads();  // the images have been read
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        float l = l_run[qt];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (g == 0) {
            ml[wave][qt * 16 + c][0] = m_run[qt];
            ml[wave][qt * 16 + c][1] = l;
        }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
            if (dt / kOwn != wave) *part_of(wave, qt, dt) = acc[qt][dt];
    }
    __syncthreads();
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
        const int r = qt * 16 + c;
        if (r >= R) continue;
        float m = ml[0][r][0], L = 0.0f, f[W];
#pragma unroll
        for (int w = 1; w < W; ++w) m = fmaxf(m, ml[w][r][0]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            f[w] = ml[w][r][0] == -INFINITY ? 0.0f : fast_exp2(ml[w][r][0] - m);
            L += ml[w][r][1] * f[w];
        }
        const int64_t orow = ((int64_t)seq * T + t_of_row[qt]) * Hq + kvh * G + (r - t_of_row[qt] * G);
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // no key seen: zeros
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            if (dt / kOwn != wave) continue;
            f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) y += (w == wave ? acc[qt][dt] : *part_of(w, qt, dt)) * f[w];
            if (num_splits == 1) {
                *reinterpret_cast<u32x2 *>(out + orow * kD + 16 * dt + 4 * g) =
                    u32x2{pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv)};
            } else {
                *reinterpret_cast<f32x4 *>(ws_o + (orow * num_splits + split) * kD + 16 * dt + 4 * g) = y;
            }
        }
        if (num_splits > 1 && wave == 0 && g == 0) {
            ws_ml[2 * (orow * num_splits + split)] = m;
            ws_ml[2 * (orow * num_splits + split) + 1] = L;
        }
    }
}

// ---------------------------------------------------------------------------
// Tile path: bf16, head_dim 128, block_size 16, any number of query rows (verify, chunked prefill).
//
// A workgroup of four waves owns a tile of the kv head's R = T * G packed query rows (row rho: new token
// rho / G, head rho % G of the group) and walks the keys in tiles of 64, two workgroups per CU:
//   KG = 1: 128 rows, 32 a wave, every wave all 64 keys;
//   KG = 2: 64 rows; waves 0, 1 take the first 32 keys of each tile and waves 2, 3 the others, so that the
//           four SIMDs share the work of few rows; the two halves join through LDS at the end.
// Codes come in as in the decode kernel, but are widened ONCE for all rows on their way into LDS
// (two buffers of K and V, one barrier a tile); two tiles are on their way, one in registers and one in LDS,
// while one is multiplied.  S^T = K Q^T and O^T = V^T P^T with mfma_f32_32x32x16: a query row lives in the lanes
// c and c + 32, P needs no lane movement.  LDS: row r, 16-byte chunk ch of K at position ch ^ (r & 15), of V
// at ch ^ 2 (r & 7) (transposed reads of 4 rows x 16 dims).
//
// Bounds: with many rows the products and, between them, the exponentials (chunk of 4 x 1024 rows behind 7168 keys,
// 2.6e11 operations: 273 to 280 us, 920 to 945 TFLOP/s); with few the loads (64 x 4096 T = 13, 537 MB: 117 us, 4.6 TB/s;
// the loads alone 110) and a workgroup's start and end (256 x 64 T = 16: 35 us of the 256 of 256 x 2048).  Two to four tiles in
// registers instead of one, three workgroups a CU, other orders of the workgroups, 8-byte staging with half the LDS
// conflicts and products interleaved with the exponentials by hand were each within 3 % or slower.
// ---------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) short s16x4;

constexpr int kWideRow = 2 * kD;              // bytes of a widened row
constexpr int kBigKeys = 64;                  // keys of a tile
constexpr int kBigBlocks = kBigKeys / kBS;
constexpr int kWideImage = kBigKeys * kWideRow;  // 16 KiB

struct Scales {  // of a tile's blocks, wave-uniform
    float k[kBigBlocks], v[kBigBlocks];
    float staged;      // V scale of the block that this wave stages
    bool large;        // lifts the reference
};

// One walk.  HALF: in f16; false, the same in all waves and with nothing written, if it met a wild scale: then the
// workgroup begins again in bf16.  (Both in one loop, as the decode kernel has them: 256 x 2048 T = 16 270 us, so 257.)
template <Kv8Format F, int KG, bool STREAM, bool HALF>
__device__ __forceinline__ bool tile_walk(
    unsigned char *lds, int &nan_seen,  // lds: [buffer][K, V]
    const __bf16 *__restrict__ q, const unsigned char *__restrict__ k_cache, const unsigned char *__restrict__ v_cache,
    const float *__restrict__ k_scales, const float *__restrict__ v_scales, const int32_t *__restrict__ block_tables,
    const int32_t *__restrict__ context_lens, __bf16 *__restrict__ out, float *__restrict__ ws_o,
    float *__restrict__ ws_ml, int T, int Hq, int Hkv, int max_blocks_per_seq, int64_t num_cache_blocks, float scale,
    int num_splits, int blocks_per_split) {
    constexpr int kRows = 128 / KG, NS = 2 / KG;  // rows of the workgroup; 32-key score tiles of a wave
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = lane >> 5, c = lane & 31;
    const int rg = KG == 1 ? wave : (wave & 1), kg = KG == 1 ? 0 : (wave >> 1);
    const int seq = blockIdx.x / Hkv, kvh = blockIdx.x % Hkv;
    const int row0 = (gridDim.y - 1 - blockIdx.y) * kRows;  // the tiles with the longest walks first
    const int split = blockIdx.z;
    const int G = Hq / Hkv, R = T * G;
    int ctx = context_lens[seq];
    const int64_t cap = (int64_t)max_blocks_per_seq * kBS;
    if (ctx > cap) ctx = (int)cap;  // never read past the table row
    if (ctx < 0) ctx = 0;
    const int row_last = row0 + kRows < R ? row0 + kRows - 1 : R - 1;
    // keys that some row of the tile sees: [0, keys); all its rows see [0, keys_all)
    const int64_t seen = (int64_t)ctx - T + row_last / G + 1;
    const int keys = seen > 0 ? (int)seen : 0;
    const int keys_all = ctx - T + row0 / G + 1;
    const int blk_begin = split * blocks_per_split;
    int blk_end = blk_begin + blocks_per_split;
    if (blk_end > (keys + kBS - 1) / kBS) blk_end = (keys + kBS - 1) / kBS;
    const int ntiles = blk_end > blk_begin ? (blk_end - blk_begin + kBigBlocks - 1) / kBigBlocks : 0;
    const int32_t *table = block_tables + (int64_t)seq * max_blocks_per_seq;

    // this lane's query row, as B operand: k-step s holds Q[row][16 s + 8 h .. + 7]
    const int row = row0 + 32 * rg + c;
    const bool live = row < R;
    const int t_row = live ? row / G : 0;
    const int64_t orow = ((int64_t)seq * T + t_row) * Hq + kvh * G + (live ? row - t_row * G : 0);
    const int last = ctx - T + t_row;  // last key it sees
    const bool works = row0 + 32 * rg < R;  // wave-uniform: waves without rows only stage
    bf16x8 qf[8];
    const unsigned flip = scale < 0.0f ? 0x80008000u : 0u;  // a negative scale moves into Q: factors stay >= 0
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        u32x4 x = {0u, 0u, 0u, 0u};
        if (live) x = *reinterpret_cast<const u32x4 *>(q + orow * kD + 16 * s + 8 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] ^= flip;
        qf[s] = __builtin_bit_cast(bf16x8, x);
    }
    const float scale_log2e = fabsf(scale) * 1.4426950408889634f;

    // staging: thread covers 16 dims (lch) of rows tid / 8 and 32 + tid / 8 of the tile
    const int64_t block_bytes = (int64_t)kBS * Hkv * kD;
    const int sr = 16 * wave + (lane >> 3), lch = threadIdx.x & 7;
    const int head_bytes = (kBS - 1) * Hkv * kD + kD;
    const unsigned lane_off = (unsigned)(sr & 15) * (unsigned)(Hkv * kD) + 16u * lch;
    const int sb = wave;  // block of the first row within its 32 keys
    unsigned kw[2], vw[2];     // LDS positions of the two 16-byte chunks of the first row; the second: + 32 rows
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        kw[e] = (unsigned)(sr * kWideRow + 16 * ((2 * lch + e) ^ (sr & 15)));
        vw[e] = (unsigned)(kWideImage + sr * kWideRow + 16 * ((2 * lch + e) ^ (2 * (sr & 7))));
    }
    Run<true> run{table, k_scales + kvh, v_scales + kvh, Hkv, blk_end, lane, num_cache_blocks};
    bool wild = false;
    auto load_tile = [&](int t, u32x4 (&ck)[2], u32x4 (&cv)[2], Scales &sc) {
        const int j = (kBigBlocks * t) & (kRun - 1);
        wild |= (run.wild >> j & ((1u << kBigBlocks) - 1)) != 0;
        sc.large = (run.large >> j & ((1u << kBigBlocks) - 1)) != 0;
        sc.staged = run.v_at(j + sb);
#pragma unroll
        for (int b = 0; b < kBigBlocks; ++b) {
            sc.k[b] = run.k_at(j + b);
            sc.v[b] = run.v_at(j + b);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t at = run.id_at(j + sb) * block_bytes + kvh * kD;
            ck[i] = load16<STREAM>(block_rows(k_cache, at, head_bytes, t < ntiles), lane_off, 8 * i * (unsigned)(Hkv * kD));
            cv[i] = load16<STREAM>(block_rows(v_cache, at, head_bytes, t < ntiles), lane_off, 8 * i * (unsigned)(Hkv * kD));
        }
        if (j == kRun - kBigBlocks) run.advance(blk_begin + kBigBlocks * (t + 1));
    };
    // codes of tile t -> bf16 (HALF: V in f16) in LDS.  V rows that no row of the tile sees are zeros, and
    // so is a NaN that only some rows see (below)
    unsigned nan_here = 0;
    auto stage_tile = [&](int t, unsigned char *buf, u32x4 (&ck)[2], u32x4 (&cv)[2], const Scales &sc) {
        const int key0 = (blk_begin + kBigBlocks * t) * kBS;
        if (key0 + kBigKeys > keys_all) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int key = key0 + 8 * i + sr;
                if (key >= keys || key >= blk_end * kBS) cv[i] = u32x4{0u, 0u, 0u, 0u};
                if constexpr (F == Kv8Format::E4M3)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const unsigned n = nan_bytes(cv[i][e]);
                        nan_here |= n;
                        cv[i][e] &= ~n;
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                *reinterpret_cast<bf16x8 *>(buf + (kw[e] ^ (i ? 128u : 0u)) + 8 * kWideRow * i) = widen8<F>(ck[i][2 * e], ck[i][2 * e + 1]);
                if constexpr (HALF)
                    *reinterpret_cast<f16x8 *>(buf + vw[e] + 8 * kWideRow * i) =
                        scaled8<F>(cv[i][2 * e], cv[i][2 * e + 1], {sc.staged, sc.staged}, {twice(sc.staged), twice(sc.staged)});
                else
                    *reinterpret_cast<bf16x8 *>(buf + vw[e] + 8 * kWideRow * i) = widen8<F>(cv[i][2 * e], cv[i][2 * e + 1]);
            }
    };

    float m_ref = -INFINITY, l_run = 0.0f;
    f32x16 acc[4];  // O^T: dims 32 dt + 8 (i / 4) + 4 h + i % 4 of this lane's row
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] = 0.0f;

    const unsigned krd = (unsigned)((32 * kg + c) * kWideRow);
    // transposed V read: lane reads 8 bytes of row 4 h + ((lane & 15) >> 2) (+ 8), dims 16 (lane >> 4 & 1) + 4 (lane & 3)
    const int vr = 4 * h + ((lane & 15) >> 2);
    const unsigned vch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const unsigned vrd = (unsigned)(kWideImage + (32 * kg + vr) * kWideRow + 8 * (lane & 1));
    auto v_fragment = [&](const unsigned char *buf, int key16, int dt) -> u32x4 {
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const unsigned at = vrd + (unsigned)(16 * key16 * kWideRow) + 16 * ((4 * dt + vch) ^ (2 * (unsigned)(vr & 7)));
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(buf + at));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(buf + at + 8 * kWideRow));
        return __builtin_bit_cast(u32x4, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    auto compute_tile = [&](int t, const unsigned char *buf, const Scales &sc) {
        const bool large = !HALF && sc.large;
        const int key0 = (blk_begin + kBigBlocks * t) * kBS + 32 * kg;
        f32x16 s[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bf16x8 a = *reinterpret_cast<const bf16x8 *>(buf + krd + 32 * kWideRow * n +
                                                                  16 * ((2 * k + h) ^ (c & 15)));
                s[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, qf[k], s[n], 0, 0, 0);
            }
        }
        // element i of score tile n is key 32 n + 8 (i / 4) + 4 h + i % 4: block 2 n + i / 8
        float f[2 * NS];
#pragma unroll
        for (int b = 0; b < 2 * NS; ++b) f[b] = (kg == 0 ? sc.k[b] : sc.k[kBigBlocks - 2 * NS + b]) * scale_log2e;
        if (key0 + 32 * NS > keys_all || key0 + 32 * NS > blk_end * kBS) {
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = key0 + 32 * n + 8 * (i / 4) + 4 * h + i % 4;
                    s[n][i] = key <= last && key < blk_end * kBS ? s[n][i] * f[2 * n + i / 8] : -INFINITY;
                }
#pragma unroll
            for (int b = 0; b < 2 * NS; ++b) f[b] = 1.0f;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2 * NS; ++b) {
            float x = s[b / 2][8 * (b % 2)];
#pragma unroll
            for (int i = 1; i < 8; ++i) x = fmaxf(x, s[b / 2][8 * (b % 2) + i]);
            mx = fmaxf(mx, x * f[b]);
        }
        mx = half_max(mx);
        if (__any(mx > m_ref + (large ? -kLift : kSlack))) {
            const float m_new = fmaxf(m_ref, mx + (large ? kLift : -kRoom));
            const float alpha = m_new == -INFINITY ? 1.0f : fast_exp2(m_ref - m_new);
            m_ref = m_new;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
        }
        const float m_safe = m_ref == -INFINITY ? 0.0f : m_ref;
        float sum = 0.0f;
        u32x4 pf[2 * NS];  // P^T as B operand, 16 keys each
#pragma unroll
        for (int b = 0; b < 2 * NS; ++b) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = fast_exp2(fmaf(s[b / 2][8 * (b % 2) + i], f[b], -m_safe));
                sum += p[i];
            }
            if constexpr (HALF) {
                pf[b] = halves(p);
            } else {
                const float v_scale = kg == 0 ? sc.v[b] : sc.v[kBigBlocks - 2 * NS + b];
#pragma unroll
                for (int i = 0; i < 8; ++i) p[i] *= v_scale;
                pf[b] = bfloats(p);
            }
        }
        l_run += sum;
#pragma unroll
        for (int b = 0; b < 2 * NS; ++b)
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                const u32x4 v = v_fragment(buf, b, dt);
                if constexpr (HALF)
                    acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), __builtin_bit_cast(f16x8, pf[b]), acc[dt], 0, 0, 0);
                else
                    acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, pf[b]), acc[dt], 0, 0, 0);
            }
        settle();
    };
    if (F == Kv8Format::E4M3 && threadIdx.x == 0) nan_seen = 0;
    if (ntiles > 0) {
        run.begin(blk_begin);
        // codes of tile t + 2 are on their way while tile t is multiplied and t + 1 goes into LDS
        u32x4 ck[2], cv[2];
        Scales sc[2];
        {
            u32x4 k0[2], v0[2];
            load_tile(0, k0, v0, sc[0]);
            load_tile(1, ck, cv, sc[1]);
            stage_tile(0, lds, k0, v0, sc[0]);
        }
        for (int t0 = 0; t0 < ntiles && !(HALF && wild); t0 += 2)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int t = t0 + u;
                __syncthreads();
                stage_tile(t + 1, lds + (1 - u) * 2 * kWideImage, ck, cv, sc[1]);
                Scales next;
                load_tile(t + 2, ck, cv, next);
                if (works && t < ntiles) compute_tile(t, lds + u * 2 * kWideImage, sc[0]);
                sc[0] = sc[1];
                sc[1] = next;
            }
    }
    if (__builtin_expect(HALF && wild, 0)) {  // all waves have seen all scales
        __syncthreads();  // the images have been read
        return false;
    }
    if constexpr (F == Kv8Format::E4M3) {
        __syncthreads();
        if (nan_here) nan_seen = 1;
        __syncthreads();
        if (nan_seen) {
            // A NaN among values that only some rows of the tile see (0 * NaN would have reached the others, so it was
            // taken for 0): which (dim, row) pairs see one is a product of zeros and ones.
            for (int t = 0; t < ntiles; ++t) {
                const int key0 = (blk_begin + kBigBlocks * t) * kBS;
                if (key0 + kBigKeys <= keys_all) continue;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int key = key0 + 8 * i + sr;
                    u32x4 one = {0u, 0u, 0u, 0u};
                    if (key < keys && key < blk_end * kBS) {
                        const int64_t at = pool_id(table[key / kBS], num_cache_blocks) * block_bytes + kvh * kD;
                        one = *reinterpret_cast<const u32x4 *>(v_cache + at + lane_off + 8 * i * (unsigned)(Hkv * kD));
#pragma unroll
                        for (int e = 0; e < 4; ++e) one[e] = nan_bytes(one[e]) & 0x38383838u;  // 1.0
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<bf16x8 *>(lds + vw[e] + 8 * kWideRow * i) = widen8<F>(one[2 * e], one[2 * e + 1]);
                }
                __syncthreads();
#pragma unroll 1
                for (int b = 0; b < 2 * NS; ++b) {
                    u32x4 see;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const int key = key0 + 32 * kg + 16 * b + 8 * (e / 4) + 4 * h + e % 4;
                        see[e / 2] = (key <= last ? 0x3f80u : 0u) | (key + 1 <= last ? 0x3f800000u : 0u);
                    }
#pragma unroll
                    for (int dt = 0; dt < 4; ++dt) {
                        f32x16 z;
#pragma unroll
                        for (int i = 0; i < 16; ++i) z[i] = 0.0f;
                        z = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v_fragment(lds, b, dt)),
                                                                    __builtin_bit_cast(bf16x8, see), z, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[dt][i] = z[i] > 0.0f ? __builtin_nanf("") : acc[dt][i];
                    }
                    settle();
                }
            }
        }
    }

    float l = half_sum(l_run);
    constexpr int kOwn = 4 / KG;  // 32-dim tiles that the wave writes
    const int dt0 = kOwn * kg;
    if constexpr (KG == 2) {
        // the two key halves' waves hand each other the dims that the other one sums, a lane's 16 bytes where the same
        // lane of the reader finds them, and (m, l)
        const auto part_of = [&](int w, int j) { return reinterpret_cast<f32x4 *>(lds + (8 * w + j) * 1024 + 16 * lane); };
        f32x2 *ml = reinterpret_cast<f32x2 *>(lds + 32 * 1024);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int q = 4 * (j & 3), d = j >> 2;
            f32x4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = kg == 0 ? acc[2 + d][q + e] : acc[d][q + e];
                acc[d][q + e] = kg == 0 ? acc[d][q + e] : acc[2 + d][q + e];  // its own dims from here on
            }
            *part_of(wave, j) = x;
        }
        ml[64 * wave + lane] = f32x2{m_ref, l};
        __syncthreads();
        const f32x2 other = ml[64 * (wave ^ 2) + lane];
        const float m = fmaxf(m_ref, other[0]);
        const float a1 = m_ref == -INFINITY ? 0.0f : fast_exp2(m_ref - m);
        const float a2 = other[0] == -INFINITY ? 0.0f : fast_exp2(other[0] - m);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const f32x4 x = *part_of(wave ^ 2, j);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                acc[j >> 2][4 * (j & 3) + e] = acc[j >> 2][4 * (j & 3) + e] * a1 + x[e] * a2;
        }
        l = l * a1 + other[1] * a2;
        m_ref = m;
    }
    if (num_splits == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
        __bf16 *op = out + orow * kD + 32 * dt0 + 8 * h;
#pragma unroll
        for (int dt = 0; dt < kOwn; ++dt)
#pragma unroll
            for (int i = 0; i < 16; i += 8) {
                // lanes c and c + 32 have dims 4 h .. + 3 of two eights: trade for one eight each
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] = __builtin_bit_cast(float, pack_bf16x2(acc[dt][i + 2 * e] * inv, acc[dt][i + 2 * e + 1] * inv));
                swap_halves(x[0], x[2]);
                swap_halves(x[1], x[3]);
                if (live)
                    *reinterpret_cast<f32x4 *>(op + 32 * dt + 2 * i) = f32x4{x[0], x[1], x[2], x[3]};
            }
    } else if (live) {
        const int64_t prow = orow * num_splits + split;
        float *op = ws_o + prow * kD + 32 * dt0 + 4 * h;
#pragma unroll
        for (int dt = 0; dt < kOwn; ++dt)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4 *>(op + 32 * dt + 2 * i) = f32x4{acc[dt][i], acc[dt][i + 1], acc[dt][i + 2], acc[dt][i + 3]};
        if (h == 0 && kg == 0) {
            ws_ml[2 * prow] = m_ref;
            ws_ml[2 * prow + 1] = l;
        }
    }
    return true;
}

template <Kv8Format F, int KG, bool STREAM>
__global__ __launch_bounds__(256, 2) void paged_attn_kv8_tile_kernel(
    const __bf16 *__restrict__ q, const unsigned char *__restrict__ k_cache, const unsigned char *__restrict__ v_cache,
    const float *__restrict__ k_scales, const float *__restrict__ v_scales, const int32_t *__restrict__ block_tables,
    const int32_t *__restrict__ context_lens, __bf16 *__restrict__ out, float *__restrict__ ws_o,
    float *__restrict__ ws_ml, int T, int Hq, int Hkv, int max_blocks_per_seq, int64_t num_cache_blocks, float scale,
    int num_splits, int blocks_per_split) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[4 * kWideImage];
    __shared__ int nan_seen;
#define NVLLM_KV8_WALK(HALF)                                                                                          \
    tile_walk<F, KG, STREAM, HALF>(lds, nan_seen, q, k_cache, v_cache, k_scales, v_scales, block_tables,             \
                                   context_lens, out, ws_o, ws_ml, T, Hq, Hkv, max_blocks_per_seq, num_cache_blocks, \
                                   scale, num_splits, blocks_per_split)
    if (!NVLLM_KV8_WALK(true)) NVLLM_KV8_WALK(false);
#undef NVLLM_KV8_WALK
}

bool fast_shape(DType dt, const PagedAttnArgs &a) {
    return dt == DType::BF16 && a.head_dim == kD && a.block_size == kBS;
}

int64_t query_rows(const PagedAttnArgs &a) { return (int64_t)a.num_new_tokens * (a.num_heads / a.num_kv_heads); }

bool decode_path(DType dt, const PagedAttnArgs &a) { return fast_shape(dt, a) && query_rows(a) <= kMaxDecodeRows; }

// workgroups of 64 rows while that is all there is, else of 128
int tile_rows(const PagedAttnArgs &a) { return query_rows(a) <= 64 ? 64 : 128; }

// Parts of the key walk: two workgroups on every CU, each part 256 keys at least.  One workgroup on every CU is more than
// half as fast as two, so with as many as that a second part pays for the merge only in longer walks (256 workgroups: 2048
// keys 51 us whole, 56 in two parts; 4096 71 and 67; 8192 137 and 126).  Fewer: 192 workgroups of 4096 keys
// 69 and 58; 64 of 4096 keys in four parts 55, whole 90.
int tile_splits(const PagedAttnArgs &a) {
    const int64_t rows = tile_rows(a);
    const int64_t units = (int64_t)a.num_seqs * a.num_kv_heads * ((query_rows(a) + rows - 1) / rows);
    const int forced = launch_policy().paged_splits;
    int64_t splits = forced > 0 ? forced : 2 * device_cus() / units;
    if (forced <= 0 && splits == 2 && a.max_blocks_per_seq < 4096 / kBS) splits = 1;
    const int64_t most = a.max_blocks_per_seq / 16;
    if (splits > most) splits = most;
    if (splits > 64) splits = 64;  // the merge kernel holds one split's (m, l) per lane
    return splits < 1 ? 1 : (int)splits;
}

// partials of a launch that is split: O and (m, l); false if the workspace is too small for them
bool partials(const PagedAttnArgs &a, int splits, float **ws_o, float **ws_ml) {
    const size_t rows = (size_t)a.num_seqs * a.num_new_tokens * a.num_heads;
    *ws_o = *ws_ml = nullptr;
    if (splits == 1) return true;
    if (!a.workspace || a.workspace_bytes < rows * splits * (kD + 2) * sizeof(float)) return false;
    *ws_o = static_cast<float *>(a.workspace);
    *ws_ml = *ws_o + rows * splits * kD;
    return true;
}

// Partials -> output, a half-wave a row, lane l dims 4 l .. + 3.
__global__ __launch_bounds__(256) void paged_attn_kv8_merge_kernel(const float *__restrict__ ws_o,
                                                                   const float *__restrict__ ws_ml,
                                                                   __bf16 *__restrict__ out, int64_t rows, int splits) {
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int l4 = 4 * (threadIdx.x & 31);
    if (row >= rows) return;
    const float *ml = ws_ml + 2 * row * splits, *o = ws_o + row * splits * kD + l4;
    float m = -INFINITY, l = 0.0f;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, ml[2 * s]);
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float w = ml[2 * s] == -INFINITY ? 0.0f : fast_exp2(ml[2 * s] - m);
        l += ml[2 * s + 1] * w;
        y += *reinterpret_cast<const f32x4 *>(o + s * kD) * w;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
    *reinterpret_cast<u32x2 *>(out + row * kD + l4) =
        u32x2{pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv)};
}

// The kernel of paged_attn.hip takes a workgroup for a row and spreads the parts over it: best for few rows or many parts
// (16384 rows of 4 parts: 19.3 us there, 7.3 here; 6656 rows of 4 9.3 and 4.9; 512 of 4 4.8 either way).
hipError_t launch_merge(const PagedAttnArgs &a, const float *ws_o, const float *ws_ml, int splits, hipStream_t stream) {
    const int64_t rows = (int64_t)a.num_seqs * a.num_new_tokens * a.num_heads;
    if (splits > 8 || rows < 1024) return launch_paged_attn_merge(ws_o, ws_ml, a.out, rows, splits, stream);
    if (rows > 8 * 0x7fffffffLL) return hipErrorInvalidValue;
    paged_attn_kv8_merge_kernel<<<dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, stream>>>(
        ws_o, ws_ml, static_cast<__bf16 *>(a.out), rows, splits);
    return hipGetLastError();
}

int blocks_per_split(const PagedAttnArgs &a, int splits, int granule) {
    const int bps = (a.max_blocks_per_seq + splits - 1) / splits;
    return (bps + granule - 1) / granule * granule;
}

// Loads that do not stay in the caches, unless what the tables reach fits the 256 MiB Infinity Cache, or other
// workgroups read the keys too (more than one tile of rows).  64 x 4096 T = 13 (512 MiB) 134 us without, 123 with; a chunk
// of 4 x 1024 rows behind 7168 keys 276 without, 281 with.
bool streams(const PagedAttnArgs &a) {
    return (int64_t)a.num_seqs * a.max_blocks_per_seq * 2 * kBS * a.num_kv_heads * kD > ((int64_t)256 << 20);
}

template <Kv8Format F, int KG, bool STREAM>
hipError_t launch_tile(const PagedAttnArgs &a, const float *ks, const float *vs, hipStream_t stream) {
    const int splits = tile_splits(a), rows = 128 / KG;
    float *ws_o, *ws_ml;
    if (!partials(a, splits, &ws_o, &ws_ml)) return hipErrorInvalidValue;
    const int64_t tiles = (query_rows(a) + rows - 1) / rows;
    if (tiles > 65535 || (int64_t)a.num_seqs * a.num_kv_heads > 0x7fffffffLL) return hipErrorInvalidValue;
    paged_attn_kv8_tile_kernel<F, KG, STREAM>
        <<<dim3((unsigned)(a.num_seqs * a.num_kv_heads), (unsigned)tiles, splits), dim3(256), 0, stream>>>(
            static_cast<const __bf16 *>(a.q), static_cast<const unsigned char *>(a.k_cache),
            static_cast<const unsigned char *>(a.v_cache), ks, vs, a.block_tables, a.context_lens,
            static_cast<__bf16 *>(a.out), ws_o, ws_ml, a.num_new_tokens, a.num_heads, a.num_kv_heads,
            a.max_blocks_per_seq, a.num_cache_blocks, a.scale, splits, blocks_per_split(a, splits, kBigBlocks));
    const hipError_t err = hipGetLastError();
    return err != hipSuccess || splits == 1 ? err : launch_merge(a, ws_o, ws_ml, splits, stream);
}

template <Kv8Format F>
hipError_t launch_tile_of(const PagedAttnArgs &a, const float *ks, const float *vs, hipStream_t stream) {
    if (tile_rows(a) != 64) return launch_tile<F, 1, false>(a, ks, vs, stream);
    return streams(a) ? launch_tile<F, 2, true>(a, ks, vs, stream) : launch_tile<F, 2, false>(a, ks, vs, stream);
}

int decode_waves(const PagedAttnArgs &a) { return query_rows(a) <= 32 ? 4 : 2; }

// Parts of the keys over workgroups: up to 1024 waves in all (4 a CU), each with 64 keys at least.  Two parts do not pay
// for the merge launch in short walks (16 x 2048: 20.8 against 20.7 us, 16 x 512 9.3 against 8.3; but 16 x 4096 T = 8 44
// whole, 33 in two), unless half the CUs would stay without the one workgroup of three query tiles that they hold.
// One query tile and long walks that the chip holds at once: parts of 2048 keys, as the last workgroups then end closer
// together (64 x 8192: 194 us whole, 177 in four parts; 32 x 16384 204 and 176; but 48 x 4096 70 and 74, 128 x 8192 with
// two rounds of workgroups 338 and 348).
int decode_splits(const PagedAttnArgs &a) {
    const int w = decode_waves(a), forced = launch_policy().paged_splits, cus = device_cus();
    const int64_t units = (int64_t)a.num_seqs * a.num_kv_heads, keys = (int64_t)a.max_blocks_per_seq * kBS;
    int64_t splits = 4 * cus / (units * w);
    if (w == 4 && splits == 2 && keys < 4096) splits = 1;
    if (query_rows(a) <= 16 && units <= 2 * cus && keys >= 8192) {
        const int64_t parts = keys / 2048 < 8 * cus / units ? keys / 2048 : 8 * cus / units;
        if (parts > splits) splits = parts;
    }
    const int64_t cap = a.max_blocks_per_seq / (4 * w);
    if (forced > 0) splits = forced;
    if (splits > cap) splits = cap;
    if (splits > 64) splits = 64;  // the merge kernel holds one split's (m, l) per lane
    return splits < 2 ? 1 : (int)splits;
}

template <Kv8Format F, int NQT, int W, bool STREAM>
void launch_decode_as(const PagedAttnArgs &a, const float *ks, const float *vs, int splits, float *ws_o, float *ws_ml,
                      hipStream_t stream) {
    paged_attn_kv8_decode_kernel<F, NQT, W, STREAM>
        <<<dim3(splits, a.num_seqs, a.num_kv_heads), dim3(64 * W), 0, stream>>>(
            static_cast<const __bf16 *>(a.q), static_cast<const unsigned char *>(a.k_cache),
            static_cast<const unsigned char *>(a.v_cache), ks, vs, a.block_tables, a.context_lens,
            static_cast<__bf16 *>(a.out), ws_o, ws_ml, a.num_new_tokens, a.num_heads, a.num_kv_heads,
            a.max_blocks_per_seq, a.num_cache_blocks, a.scale, splits, blocks_per_split(a, splits, kTileBlocks));
}

template <Kv8Format F>
hipError_t launch_decode(const PagedAttnArgs &a, const float *ks, const float *vs, hipStream_t stream) {
    const int splits = decode_splits(a);
    float *ws_o, *ws_ml;
    if (!partials(a, splits, &ws_o, &ws_ml)) return hipErrorInvalidValue;
    const bool nt = streams(a);
#define NVLLM_KV8_CASE(NQT, W)                                                                  \
    case NQT:                                                                                   \
        if (nt) launch_decode_as<F, NQT, W, true>(a, ks, vs, splits, ws_o, ws_ml, stream);      \
        else launch_decode_as<F, NQT, W, false>(a, ks, vs, splits, ws_o, ws_ml, stream);        \
        break;
    switch ((int)((query_rows(a) + 15) / 16)) {
        NVLLM_KV8_CASE(1, 4) NVLLM_KV8_CASE(2, 4) NVLLM_KV8_CASE(3, 2)
        default: return hipErrorInvalidValue;
    }
#undef NVLLM_KV8_CASE
    const hipError_t err = hipGetLastError();
    return err != hipSuccess || splits == 1 ? err : launch_merge(a, ws_o, ws_ml, splits, stream);
}

int splits_of(DType dt, const PagedAttnArgs &a) {
    if (!fast_shape(dt, a)) return 1;
    return decode_path(dt, a) ? decode_splits(a) : tile_splits(a);
}

}  // namespace

PagedKv8Path paged_attn_kv8_path(DType dt, const PagedAttnArgs &a) {
    if (!fast_shape(dt, a)) return PagedKv8Path::Generic;
    return decode_path(dt, a) ? PagedKv8Path::Decode : PagedKv8Path::Tile;
}

size_t paged_attn_kv8_workspace_bytes(DType dt, const PagedAttnArgs &a) {
    const int splits = splits_of(dt, a);
    if (splits <= 1) return 0;
    return (size_t)a.num_seqs * a.num_new_tokens * a.num_heads * splits * (kD + 2) * sizeof(float);
}

hipError_t launch_paged_attn_kv8(DType dt, Kv8Format fmt, const PagedAttnArgs &a, const float *k_scales,
                                 const float *v_scales, hipStream_t stream) {
    if (a.num_seqs <= 0) return hipSuccess;
    const bool int8 = fmt == Kv8Format::Int8;
    if (decode_path(dt, a))
        return int8 ? launch_decode<Kv8Format::Int8>(a, k_scales, v_scales, stream)
                    : launch_decode<Kv8Format::E4M3>(a, k_scales, v_scales, stream);
    if (fast_shape(dt, a)) {
        return int8 ? launch_tile_of<Kv8Format::Int8>(a, k_scales, v_scales, stream)
                    : launch_tile_of<Kv8Format::E4M3>(a, k_scales, v_scales, stream);
    }
    if (dt == DType::BF16)
        return fmt == Kv8Format::Int8 ? launch_generic<__bf16, Kv8Format::Int8>(a, k_scales, v_scales, stream)
                                      : launch_generic<__bf16, Kv8Format::E4M3>(a, k_scales, v_scales, stream);
    return fmt == Kv8Format::Int8 ? launch_generic<float, Kv8Format::Int8>(a, k_scales, v_scales, stream)
                                  : launch_generic<float, Kv8Format::E4M3>(a, k_scales, v_scales, stream);
}

}  // namespace kernels
}  // namespace nvllm

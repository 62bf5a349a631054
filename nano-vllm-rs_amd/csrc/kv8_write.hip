// kv8_write.hip -- writing and reading the 8-bit KV cache (gfx950): the quantising forms of
// reshape_and_cache (K4), of the producer (K5), and of the block gather.
//
// The number formats and the scale's formula are in kv8_common.hpp.  What a write does to a block:
// let W be the rows (slots of the block) that the call writes and need = scale_of(max |x| over W).
//   W holds the block's row 0:  scale' = need.  The block begins; what it held is gone.
//   otherwise:                  scale' = max(scale, need).  If that grew, the codes of the rows not
//                               in W are rounded to the new scale.
//   code(x) = round(x / scale') for the rows in W.
// Blocks are filled in order (BlockTable::get_slot_mapping, reference src/core/block.rs:269-283), so
// row 0 is written exactly when a block comes fresh from the allocator: no call has to reset scales.
//
// The scale couples all tokens that a call puts into one block, and a slot mapping may name them in
// any order.  So each block gets ONE owner: the workgroup that looks after the first of its tokens.  It
// finds the block's other tokens, takes the maximum, and writes codes and scale; no atomics on the cache, and of tokens that name the same slot the last one wins, as in a sequential
// loop (the reference's, src/attention/paged.rs:231-262).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "kv8_common.hpp"

namespace nvllm {
namespace kernels {

namespace {

using namespace kv8;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxChunk = 16;  // tokens a workgroup looks after

// Up to this many tokens every workgroup reads the whole slot mapping to find its blocks' tokens;
// above, a launch in front leaves slot -> token in the workspace.  (Scanned against indexed, us: prompts of 256 7.1 and
// 8.4, 1024 9.0 and 9.7, 2048 11.2 and 11.2, 4096 14.0 and 12.0; decode steps of 1024 8.6 and 8.5, of 2048 12.0 and 9.2.)
constexpr int64_t kScanTokens = 1024;

// slot -> token for every slot the call writes.  Nothing is cleared first: an entry counts only if
// the token it names writes that very slot, so whatever else the workspace holds is seen through.
// The last token that names a slot wins, by compare-and-swap.
__global__ __launch_bounds__(kThreads) void kv8_index_kernel(const int64_t *__restrict__ slots, int n,
                                                             int64_t num_slots, int32_t *index) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    const int t = (int)i;
    const int64_t s = slots[t];
    if (s < 0 || s >= num_slots) return;
    int seen = index[s];
    while (!(seen >= t && seen < n && slots[seen] == s)) {
        const int was = atomicCAS(index + s, seen, t);
        if (was == seen) break;
        seen = was;
    }
}

// The blocks that this chunk of tokens owns: those whose first token (of the tokens whose row is not
// overwritten by a later one) is in the chunk.  LDS: map[u * bs + o] = the token of the call that writes row
// o of the chunk's u-th block (-1: none).  Returns how many blocks the chunk owns, owner[i] = u of the i-th.
struct Chunk {
    int *map;      // [kMaxChunk * bs]
    int *owner;    // [kMaxChunk]
    int *block;    // [kMaxChunk]: the different blocks of the chunk's slots
    int *rows;     // [kMaxChunk + 1] or none: rows of the u-th block, if the call writes one (o | 0xff00) or two
                   // (o | o' << 8) of them, else -1; and how many of the chunk's own blocks those are
};

__device__ __forceinline__ int find_blocks(const Chunk &ch, const int64_t *__restrict__ slots, int n, int t0,
                                           int chunk, int bs, int64_t num_slots,
                                           const int32_t *__restrict__ index) {
    __shared__ int uniques, count;
    const int tid = threadIdx.x;
    if (tid < 64) {
        int b = -1;
        if (tid < chunk && t0 + tid < n) {
            const int64_t s = slots[t0 + tid];
            if (s >= 0 && s < num_slots) b = (int)(s / bs);
        }
        bool first = b >= 0;
        for (int j = 0; j < chunk - 1; ++j) {
            const int bj = __shfl(b, j);  // by all lanes: an inactive one has nothing to read
            if (j < tid && bj == b) first = false;
        }
        const unsigned long long m = __ballot(first);
        if (first) ch.block[__popcll(m & ((1ull << tid) - 1))] = b;
        if (tid == 0) uniques = __popcll(m);
    }
    __syncthreads();
    const int nu = uniques;
    if (index) {
        for (int i = tid; i < nu * bs; i += kThreads) {
            const int64_t s = (int64_t)ch.block[i / bs] * bs + i % bs;
            int e = index[s];
            if (e < 0 || e >= n || slots[e] != s) e = -1;
            ch.map[i] = e;
        }
    } else {
        for (int i = tid; i < nu * bs; i += kThreads) ch.map[i] = -1;
        __syncthreads();
        for (int t = tid; t < n; t += kThreads) {
            const int64_t s = slots[t];
            if (s < 0 || s >= num_slots) continue;
            const int b = (int)(s / bs);
            for (int u = 0; u < nu; ++u)
                if (ch.block[u] == b) atomicMax(ch.map + u * bs + (int)(s - (int64_t)b * bs), t);
        }
    }
    __syncthreads();
    if (tid < 64) {
        int first = n, some = 0xffff, many = 0;
        for (int o = 0; tid < nu && o < bs; ++o) {
            const int t = ch.map[tid * bs + o];
            if (t < 0) continue;
            if (t < first) first = t;
            if (++many <= 2) some = many == 1 ? 0xff00 | o : (some & 255) | o << 8;
        }
        if (ch.rows && tid < nu) ch.rows[tid] = many <= 2 ? some : -1;
        const bool mine = tid < nu && first >= t0 && first < t0 + chunk;
        const unsigned long long m = __ballot(mine);  // the same order in every workgroup that looks after the chunk
        if (mine) ch.owner[__popcll(m & ((1ull << tid) - 1))] = tid;
        const unsigned long long f = __ballot(mine && many <= 2);
        if (tid == 0) {
            count = __popcll(m);
            if (ch.rows) ch.rows[kMaxChunk] = __popcll(f);
        }
    }
    __syncthreads();
    return count;
}

// Scale and codes of one (block, kv head) of K or V by one wave, any head_dim and block_size.
// row(t) is called by the whole wave and returns a functor d -> value of token t's row.
template <Kv8Format F, typename Row>
__device__ __forceinline__ void write_unit(const int *map, int bs, int D, int Hkv, int64_t block, int head,
                                           unsigned char *cache, float *scales, const Row &row) {
    const int lane = threadIdx.x & 63;
    float amax = 0.0f;
    for (int o = 0; o < bs; ++o) {
        const int t = map[o];
        if (t < 0) continue;
        const auto x = row(t);
        for (int d = lane; d < D; d += 64) amax = fmaxf(amax, finite_abs(narrow_odd(x(d))));  // past a border stays past it
    }
    const float need = scale_of<F>(wave_max(amax));
    const bool begins = map[0] >= 0;
    float *sp = scales + block * Hkv + head;
    const float was = begins ? 0.0f : *sp;
    const float s = fmaxf(was, need);
    const float inv = inverse_scale(s);
    unsigned char *base = cache + (block * bs * Hkv + head) * (int64_t)D;
    for (int o = 0; o < bs; ++o) {
        unsigned char *out = base + (int64_t)o * Hkv * D;
        const int t = map[o];
        if (t >= 0) {
            const auto x = row(t);
            for (int d = lane; d < D; d += 64) out[d] = encode1<F>(x(d) * inv);
        } else if (!begins && s > was) {
            const float ratio = was * inv;
            for (int d = lane; d < D; d += 64) out[d] = (unsigned char)rescale4<F>(out[d], ratio);
        }
    }
    if (lane == 0 && (begins || s > was)) *sp = s;
}

// Norm and rotation of one row by one wave: x / sqrt(mean(x^2) + eps) * weight, then the rotation of
// the pairs (d, d + D/2).  AT: f64 for what is quantised, as a value that f32 arithmetic moves across a code's
// border would show as a whole step (and f64 runs at the rate of f32 here); f32 for what is not.
template <typename ET, typename AT> struct RotatedRow {
    const ET *x, *w, *c, *s;
    int half;
    AT inv;
    __device__ __forceinline__ AT operator()(int d) const {
        const int lo = d < half ? d : d - half;
        const AT a = (AT)to_f32(x[lo]) * inv * (AT)to_f32(w[lo]);
        const AT b = (AT)to_f32(x[lo + half]) * inv * (AT)to_f32(w[lo + half]);
        return d < half ? a * (AT)to_f32(c[d]) - b * (AT)to_f32(s[d]) : b * (AT)to_f32(c[d]) + a * (AT)to_f32(s[d]);
    }
};

template <typename ET, typename AT>
__device__ __forceinline__ RotatedRow<ET, AT> rotated_row(const ET *x, const ET *w, const ET *cos_cache,
                                                          const ET *sin_cache, int pos, int max_pos, int D, float eps) {
    const int lane = threadIdx.x & 63;
    pos = pos < 0 ? 0 : (pos >= max_pos ? max_pos - 1 : pos);  // never read outside the tables
    AT ss = 0;
    for (int d = lane; d < D; d += 64) ss += (AT)to_f32(x[d]) * (AT)to_f32(x[d]);
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) ss += __shfl_xor(ss, m);
    return {x, w, cos_cache + (int64_t)pos * D, sin_cache + (int64_t)pos * D, D / 2,
            (AT)1 / (AT)sqrt((AT)(ss / (AT)D + (AT)eps))};
}

template <typename ET> struct PlainRow {
    const ET *x;
    __device__ __forceinline__ float operator()(int d) const { return to_f32(x[d]); }
};

// Any head_dim and block_size.  Workgroups [0, row_blocks) normalise and rotate rows of Q (and of K
// to k_out, if asked), one a wave; the rest look after `chunk` tokens' cache blocks each.
template <typename ET, Kv8Format F, bool PRODUCER>
__global__ __launch_bounds__(kThreads) void kv8_write_generic_kernel(const Kv8WriteArgs a, int chunk, int row_blocks,
                                                                     bool indexed) {
    typedef typename std::conditional<sizeof(ET) == 4, double, float>::type QT;  // of q_out and k_out
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int D = a.head_dim, Hkv = a.num_kv_heads, Hq = a.num_heads;
    const ET *key = static_cast<const ET *>(a.key), *value = static_cast<const ET *>(a.value);
    if constexpr (PRODUCER) {
        if ((int)blockIdx.x < row_blocks) {
            const int heads = Hq + (a.k_out ? Hkv : 0);
            const int64_t r = (int64_t)blockIdx.x * kWaves + wave;
            const int64_t t = r / heads;
            if (t >= a.num_tokens) return;
            const int h = (int)(r - t * heads);
            const ET *x = h < Hq ? static_cast<const ET *>(a.q) + (t * Hq + h) * D : key + (t * Hkv + h - Hq) * D;
            ET *y = h < Hq ? static_cast<ET *>(a.q_out) + (t * Hq + h) * D
                           : static_cast<ET *>(a.k_out) + (t * Hkv + h - Hq) * D;
            const auto row = rotated_row<ET, QT>(x, static_cast<const ET *>(h < Hq ? a.q_weight : a.k_weight),
                                                 static_cast<const ET *>(a.cos_cache),
                                                 static_cast<const ET *>(a.sin_cache), a.positions[t], a.max_positions,
                                                 D, a.eps);
            for (int d = lane; d < D / 2; d += 64) {  // both of a pair are read before either is written: y may be x
                const ET lo = static_cast<ET>((float)row(d)), hi = static_cast<ET>((float)row(d + D / 2));
                y[d] = lo;
                y[d + D / 2] = hi;
            }
            return;
        }
    }
    extern __shared__ int dyn[];
    __shared__ int owner[kMaxChunk];
    __shared__ int block[kMaxChunk];
    const Chunk ch{dyn, owner, block, nullptr};
    const int bs = a.block_size, n = (int)a.num_tokens, t0 = ((int)blockIdx.x - row_blocks) * chunk;
    const int count = find_blocks(ch, a.slot_mapping, n, t0, chunk, bs, a.num_cache_blocks * bs,
                                  indexed ? a.workspace : nullptr);
    for (int u = wave; u < count * Hkv * 2; u += kWaves) {
        const int i = u / (2 * Hkv), head = u % Hkv;
        const bool is_v = (u / Hkv) & 1;
        const int c = owner[i];
        const int *map = dyn + c * bs;
        unsigned char *cache = static_cast<unsigned char *>(is_v ? a.v_cache : a.k_cache);
        float *scales = is_v ? a.v_scales : a.k_scales;
        if (PRODUCER && !is_v)
            write_unit<F>(map, bs, D, Hkv, block[c], head, cache, scales, [&](int t) {
                return rotated_row<ET, double>(key + ((int64_t)t * Hkv + head) * D, static_cast<const ET *>(a.k_weight),
                                           static_cast<const ET *>(a.cos_cache), static_cast<const ET *>(a.sin_cache),
                                           a.positions[t], a.max_positions, D, a.eps);
            });
        else
            write_unit<F>(map, bs, D, Hkv, block[c], head, cache, scales, [&](int t) {
                return PlainRow<ET>{(is_v ? value : key) + ((int64_t)t * Hkv + head) * D};
            });
    }
}

template <typename ET, Kv8Format F>
hipError_t launch_generic(const Kv8WriteArgs &a, bool indexed, hipStream_t stream) {
    int chunk = kMaxChunk;
    while (chunk > 1 && a.num_tokens / chunk < 512) chunk /= 2;
    const int64_t chunks = (a.num_tokens + chunk - 1) / chunk;
    const size_t lds = (size_t)chunk * a.block_size * sizeof(int);
    if (a.q) {
        const int64_t rows = a.num_tokens * (a.num_heads + (a.k_out ? a.num_kv_heads : 0));
        const int64_t row_blocks = (rows + kWaves - 1) / kWaves;
        if (row_blocks + chunks > 0x7fffffffLL) return hipErrorInvalidValue;
        kv8_write_generic_kernel<ET, F, true><<<dim3((unsigned)(row_blocks + chunks)), dim3(kThreads), lds, stream>>>(
            a, chunk, (int)row_blocks, indexed);
    } else {
        kv8_write_generic_kernel<ET, F, false><<<dim3((unsigned)chunks), dim3(kThreads), lds, stream>>>(a, chunk, 0,
                                                                                                     indexed);
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Fast path: bf16, head_dim 128, block_size 16.
//
// Bound by HBM on prompts (K and V read once, half as many bytes written) and by latency on a decode step.
// A wave takes one (block, kv head) of K or V: 8 lanes a row, two rows a lane (o and o + 8), so the block is
// read with four 16-byte loads a lane, its maximum found with six shuffles and written with two 16-byte
// stores, all rows of the block at once.  Of a block that gets one or two rows (a decode step) a wave takes
// eight heads instead, 8 lanes those of one head: the producer's decode step of 256 (32 and 8 heads) 10.3 -> 7.3
// us, of 1024 28.2 -> 12.5 (in a kernel trace).  `parts` workgroups share a chunk's units, so that few tokens still spread over the chip.
// ---------------------------------------------------------------------------
constexpr int kFastD = 128;
constexpr int kFastBS = 16;

// 16 values of a row.  Plain rows: dims 16 ch .. + 15.  Rotated rows: 8 ch .. + 7, then 64 + 8 ch .. + 7, so
// that a lane holds both dims of its pairs.
template <bool ROT> __device__ __forceinline__ int dim_of(int ch, int half) {
    return ROT ? 64 * half + 8 * ch : 16 * ch + 8 * half;
}

__device__ __forceinline__ void unpack8(u32x4 w, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = bf16_lo(w[i]);
        x[2 * i + 1] = bf16_hi(w[i]);
    }
}

// Norm and rotation of a row that 8 lanes hold (lo: dims 8 ch .. + 7, hi: 64 + 8 ch ..; y[0 .. 7], y[8 .. 15]), in AT;
// in f32, f64 results are rounded to odd.
template <typename AT>
__device__ __forceinline__ void rotate_row(u32x4 lo, u32x4 hi, const __bf16 *w, const __bf16 *cos_row,
                                           const __bf16 *sin_row, int ch, float eps, float *y) {
    const auto get = [&](const __bf16 *p, u32x4 &l, u32x4 &h) {
        l = *reinterpret_cast<const u32x4 *>(p + 8 * ch);
        h = *reinterpret_cast<const u32x4 *>(p + 64 + 8 * ch);
    };
    u32x4 w1, w2, c1, c2, s1, s2;
    get(cos_row, c1, c2);
    get(sin_row, s1, s2);
    get(w, w1, w2);
    const auto at = [](u32x4 p, int i) -> AT { return (AT)(i & 1 ? bf16_hi(p[i / 2]) : bf16_lo(p[i / 2])); };
    AT ss = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += at(lo, i) * at(lo, i) + at(hi, i) * at(hi, i);
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) ss += __shfl_xor(ss, m);
    const AT inv = (AT)1 / (AT)sqrt((AT)(ss * (AT)(1.0 / kFastD) + (AT)eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const AT n1 = at(lo, i) * inv * at(w1, i), n2 = at(hi, i) * inv * at(w2, i);
        y[i] = narrow_odd(n1 * at(c1, i) - n2 * at(s1, i));
        y[8 + i] = narrow_odd(n2 * at(c2, i) + n1 * at(s2, i));
    }
}

// FEW: a block of which the call writes one or two rows (`rows`: which).  8 lanes then take those of one head, and the
// wave eight heads from `head0` on.
template <Kv8Format F, bool ROT, bool FEW>
__device__ __forceinline__ void write_fast_unit(const Kv8WriteArgs &a, const int *map, int rows, int block, int head0,
                                                bool is_v) {
    const int lane = threadIdx.x & 63, r = lane >> 3, ch = lane & 7;
    const int Hkv = a.num_kv_heads, head = FEW ? head0 + r : head0;
    const bool valid = !FEW || head < Hkv;
    const __bf16 *src = static_cast<const __bf16 *>(is_v ? a.value : a.key);
    float *sp = (is_v ? a.v_scales : a.k_scales) + (int64_t)block * Hkv + head;
    const bool begins = map[0] >= 0;
    const float was = begins || !valid ? 0.0f : *sp;
    u32x4 w[2][2];
    int o[2], t[2], pos[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        o[i] = FEW ? rows >> (8 * i) & 255 : r + 8 * i;
        t[i] = valid && o[i] < kFastBS ? map[o[i]] : -1;
        pos[i] = 0;
        w[i][0] = w[i][1] = u32x4{0u, 0u, 0u, 0u};
        if (t[i] >= 0) {
            if constexpr (ROT) pos[i] = a.positions[t[i]];
            const __bf16 *p = src + ((int64_t)t[i] * Hkv + head) * kFastD;
            w[i][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + dim_of<ROT>(ch, 0)));
            w[i][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + dim_of<ROT>(ch, 1)));
        }
    }
    float x[2][16];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (ROT) {
#pragma unroll
            for (int j = 0; j < 16; ++j) x[i][j] = 0.0f;
            if (__any(t[i] >= 0)) {  // a decode step writes one row of a block
                const int at = pos[i] < 0 ? 0 : (pos[i] >= a.max_positions ? a.max_positions - 1 : pos[i]);  // inside the tables
                rotate_row<double>(w[i][0], w[i][1], static_cast<const __bf16 *>(a.k_weight),
                                   static_cast<const __bf16 *>(a.cos_cache) + (int64_t)at * kFastD,
                                   static_cast<const __bf16 *>(a.sin_cache) + (int64_t)at * kFastD, ch, a.eps, x[i]);
                if (t[i] < 0)  // a row of zeros with eps 0 is NaN here
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[i][j] = 0.0f;
            }
            __builtin_amdgcn_sched_barrier(0);  // one row after the other: both at once take 170 registers
        } else {
            unpack8(w[i][0], x[i]);
            unpack8(w[i][1], x[i] + 8);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) amax = fmaxf(amax, finite_abs(x[i][j]));
    }
    if constexpr (FEW) {
#pragma unroll
        for (int m = 1; m < 8; m <<= 1) amax = fmaxf(amax, __shfl_xor(amax, m));
    } else {
        amax = wave_max(amax);
    }
    const float s = fmaxf(was, scale_of<F>(amax));
    const float inv = inverse_scale(s), ratio = was * inv;
    const bool grows = !begins && s > was;
    unsigned char *base = static_cast<unsigned char *>(is_v ? a.v_cache : a.k_cache) +
                          ((int64_t)block * kFastBS * Hkv + head) * kFastD;
    const auto rescale = [&](int row) {
        u32x4 *out = reinterpret_cast<u32x4 *>(base + (int64_t)row * Hkv * kFastD + 16 * ch);
        u32x4 y = *out;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = rescale4<F>(y[j], ratio);
        *out = y;
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        unsigned char *out = base + (int64_t)o[i] * Hkv * kFastD;
        unsigned c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            c[j] = encode4<F>(x[i][4 * j] * inv, x[i][4 * j + 1] * inv, x[i][4 * j + 2] * inv, x[i][4 * j + 3] * inv);
        if constexpr (ROT) {
            // even lanes have dims 8 ch and 64 + 8 ch; trade with the neighbour for 16 dims in a row:
            // even lanes 8 ch .. + 15, odd lanes 64 + 8 (ch - 1) .. + 15
            const bool odd = ch & 1;
            const unsigned g0 = __shfl_xor((int)(odd ? c[0] : c[2]), 1), g1 = __shfl_xor((int)(odd ? c[1] : c[3]), 1);
            const u32x4 y = odd ? u32x4{g0, g1, c[2], c[3]} : u32x4{c[0], c[1], g0, g1};
            if (t[i] >= 0) *reinterpret_cast<u32x4 *>(out + (odd ? 64 + 8 * (ch - 1) : 8 * ch)) = y;
        } else {
            if (t[i] >= 0) *reinterpret_cast<u32x4 *>(out + 16 * ch) = u32x4{c[0], c[1], c[2], c[3]};
        }
        if constexpr (!FEW)
            if (grows && t[i] < 0) rescale(o[i]);
    }
    if constexpr (FEW)
        if (grows)
            for (int row = 0; row < kFastBS; ++row)
                if (row != o[0] && row != o[1]) rescale(row);
    if ((FEW ? ch == 0 && valid : lane == 0) && (begins || grows)) *sp = s;
}

// Workgroups [0, chunk_blocks * parts): part `% parts` of chunk `/ parts`; behind them (producer) rows of Q, and of
// K to k_out, 8 lanes a row, 32 rows a workgroup.  Waves a SIMD: 8 for the plain write (8 x 4096 tokens 42.6 us, with 7
// 44.8), 4 for the producer with its f64 rows (3: 4 x 2048 tokens 33.5 us against 31; 5 spill).
template <Kv8Format F, bool PRODUCER>
__global__ __launch_bounds__(kThreads, PRODUCER ? 4 : 8) void kv8_write_kernel(const Kv8WriteArgs a, int chunk,
                                                                              int parts, int chunk_blocks, bool indexed) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int Hkv = a.num_kv_heads;
    if constexpr (PRODUCER) {
        if (blockIdx.x >= (unsigned)(chunk_blocks * parts)) {
            const int Hq = a.num_heads, heads = Hq + (a.k_out ? Hkv : 0);
            const int64_t rows = a.num_tokens * heads;
            const int64_t r = (int64_t)(blockIdx.x - chunk_blocks * parts) * 32 + (threadIdx.x >> 3);
            if (r >= rows) return;  // whole groups of 8 lanes leave together
            const int64_t t = rows <= 0xffffffffLL ? (int64_t)((unsigned)r / (unsigned)heads) : r / heads;
            const int h = (int)(r - t * heads), ch = threadIdx.x & 7;
            const bool is_q = h < Hq;
            const int64_t at = is_q ? (t * Hq + h) * kFastD : (t * Hkv + h - Hq) * kFastD;
            const __bf16 *p = static_cast<const __bf16 *>(is_q ? a.q : a.key) + at;
            __bf16 *y = static_cast<__bf16 *>(is_q ? a.q_out : a.k_out) + at;
            int pos = a.positions[t];
            pos = pos < 0 ? 0 : (pos >= a.max_positions ? a.max_positions - 1 : pos);
            float x[16];
            rotate_row<float>(__builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + 8 * ch)),
                              __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + 64 + 8 * ch)),
                              static_cast<const __bf16 *>(is_q ? a.q_weight : a.k_weight),
                              static_cast<const __bf16 *>(a.cos_cache) + (int64_t)pos * kFastD,
                              static_cast<const __bf16 *>(a.sin_cache) + (int64_t)pos * kFastD, ch, a.eps, x);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                *reinterpret_cast<u32x4 *>(y + 64 * i + 8 * ch) =
                    u32x4{pack_bf16x2(x[8 * i], x[8 * i + 1]), pack_bf16x2(x[8 * i + 2], x[8 * i + 3]),
                          pack_bf16x2(x[8 * i + 4], x[8 * i + 5]), pack_bf16x2(x[8 * i + 6], x[8 * i + 7])};
            return;
        }
    }
    __shared__ int map[kMaxChunk * kFastBS], owner[kMaxChunk], block[kMaxChunk], rows[kMaxChunk + 1];
    const Chunk ch{map, owner, block, rows};
    const int part = blockIdx.x % parts, t0 = (int)(blockIdx.x / parts) * chunk;
    const int count = find_blocks(ch, a.slot_mapping, (int)a.num_tokens, t0, chunk, kFastBS,
                                  a.num_cache_blocks * kFastBS, indexed ? a.workspace : nullptr);
    const int first = part * kWaves + wave, stride = parts * kWaves, eights = (Hkv + 7) / 8;
    const int fews = __builtin_amdgcn_readfirstlane(rows[kMaxChunk]);
    if (fews > 0)
        for (int u = first; u < count * eights * 2; u += stride) {
            const int i = u / (2 * eights), c = __builtin_amdgcn_readfirstlane(owner[i]);
            const int b = __builtin_amdgcn_readfirstlane(block[c]), few = __builtin_amdgcn_readfirstlane(rows[c]);
            const bool is_v = (u / eights) & 1;
            if (few < 0) continue;
            if (PRODUCER && !is_v)
                write_fast_unit<F, true, true>(a, map + c * kFastBS, few, b, 8 * (u % eights), false);
            else
                write_fast_unit<F, false, true>(a, map + c * kFastBS, few, b, 8 * (u % eights), is_v);
        }
    if (fews < count)
        for (int u = first; u < count * Hkv * 2; u += stride) {
            const int i = u / (2 * Hkv), c = __builtin_amdgcn_readfirstlane(owner[i]);
            const int b = __builtin_amdgcn_readfirstlane(block[c]), few = __builtin_amdgcn_readfirstlane(rows[c]);
            const bool is_v = (u / Hkv) & 1;
            if (few >= 0) continue;
            if (PRODUCER && !is_v)
                write_fast_unit<F, true, false>(a, map + c * kFastBS, 0, b, u % Hkv, false);
            else
                write_fast_unit<F, false, false>(a, map + c * kFastBS, 0, b, u % Hkv, is_v);
        }
}

template <Kv8Format F> hipError_t launch_fast(const Kv8WriteArgs &a, bool indexed, hipStream_t stream) {
    // tokens per workgroup: up to a block's worth, while that leaves work for every CU
    int chunk = kMaxChunk;
    while (chunk > 1 && a.num_tokens < (int64_t)chunk * 256) chunk /= 2;
    const int64_t chunks = (a.num_tokens + chunk - 1) / chunk;
    // workgroups per chunk: a unit a wave while the launch is small; the producer's leave some of the chip's 1024 places
    // to the rows of Q (4 x 2048 tokens: 31 us, 38 with up to 2048 of them)
    int parts = (2 * a.num_kv_heads + kWaves - 1) / kWaves;
    while (parts > 1 && chunks * parts > (a.q ? 768 : 2048)) --parts;
    const int64_t rows = a.q ? a.num_tokens * (a.num_heads + (a.k_out ? a.num_kv_heads : 0)) : 0;
    const int64_t blocks = chunks * parts + (rows + 31) / 32;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (a.q)
        kv8_write_kernel<F, true><<<dim3((unsigned)blocks), dim3(kThreads), 0, stream>>>(a, chunk, parts, (int)chunks, indexed);
    else
        kv8_write_kernel<F, false><<<dim3((unsigned)blocks), dim3(kThreads), 0, stream>>>(a, chunk, parts, (int)chunks, indexed);
    return hipGetLastError();
}

bool fast_shape(DType dt, const Kv8WriteArgs &a) {
    const auto at16 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    return dt == DType::BF16 && a.head_dim == kFastD && a.block_size == kFastBS && at16(a.key) && at16(a.value) &&
           at16(a.k_cache) && at16(a.v_cache) && at16(a.q) && at16(a.q_out) && at16(a.k_out) && at16(a.q_weight) &&
           at16(a.k_weight) && at16(a.cos_cache) && at16(a.sin_cache);
}

// Read-back of whole blocks: out[i] = codes of block ids[i] times its scales, in bf16 or f32 (exact where the type has the number).
// Eight values a thread (D a multiple of 8), else one; blockIdx.y takes K and V.
// Ids outside the pool give zeros.
template <typename ET, Kv8Format F, int V>
__global__ __launch_bounds__(256) void kv8_gather_kernel(const unsigned char *__restrict__ k_cache,
                                                         const unsigned char *__restrict__ v_cache,
                                                         const float *__restrict__ k_scales,
                                                         const float *__restrict__ v_scales,
                                                         const int32_t *__restrict__ ids, ET *__restrict__ k_out,
                                                         ET *__restrict__ v_out, int64_t total, int block_vec,
                                                         int Hkv, int D, int64_t num_cache_blocks) {
    const int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (g >= total) return;
    const bool is_v = blockIdx.y;
    const unsigned char *cache = is_v ? v_cache : k_cache;
    ET *out = (is_v ? v_out : k_out) + g * V;
    const int64_t i = total <= 0xffffffffLL ? (int64_t)((unsigned)g / (unsigned)block_vec) : g / block_vec;
    const int idx = (int)(g - i * block_vec) * V;
    const int64_t id = ids[i];
    float x[V];
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = 0.0f;
    if (id >= 0 && id < num_cache_blocks) {
        const float s = (is_v ? v_scales : k_scales)[id * Hkv + (idx / D) % Hkv];
        const unsigned char *p = cache + id * ((int64_t)block_vec * V) + idx;
        if constexpr (V == 8) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(p);
            decode4<F>(w[0], x);
            decode4<F>(w[1], x + 4);
        } else {
            x[0] = decode1<F>(*p);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] *= s;
    }
    if constexpr (V == 8 && sizeof(ET) == 2) {
        const u32x4 y = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                         pack_bf16x2(x[6], x[7])};
        __builtin_nontemporal_store(y, reinterpret_cast<u32x4 *>(out));
    } else if constexpr (V == 8) {
        __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4 *>(out));
        __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, reinterpret_cast<f32x4 *>(out) + 1);
    } else {
        *out = static_cast<ET>(x[0]);
    }
}

template <typename ET, Kv8Format F, int V>
hipError_t launch_gather(const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales,
                         const int32_t *ids, int64_t num_ids, void *k_out, void *v_out, int64_t num_cache_blocks,
                         int block_size, int Hkv, int D, hipStream_t stream) {
    const int64_t vec = (int64_t)block_size * Hkv * D / V, total = num_ids * vec, blocks = (total + 255) / 256;
    if (vec * V > 0x7fffffffLL || blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    kv8_gather_kernel<ET, F, V><<<dim3((unsigned)blocks, v_out ? 2 : 1), dim3(256), 0, stream>>>(
        static_cast<const unsigned char *>(k_cache), static_cast<const unsigned char *>(v_cache), k_scales, v_scales,
        ids, static_cast<ET *>(k_out), static_cast<ET *>(v_out), total, (int)vec, Hkv, D, num_cache_blocks);
    return hipGetLastError();
}

}  // namespace

size_t kv8_write_workspace_bytes(int64_t num_tokens, int block_size, int64_t num_cache_blocks) {
    return num_tokens > kScanTokens ? (size_t)num_cache_blocks * block_size * sizeof(int32_t) : 0;
}

hipError_t launch_kv8_write(DType dt, Kv8Format fmt, const Kv8WriteArgs &a, hipStream_t stream) {
    if (a.num_tokens <= 0) return hipSuccess;
    const bool indexed = kv8_write_workspace_bytes(a.num_tokens, a.block_size, a.num_cache_blocks) > 0;
    if (indexed) {
        if (!a.workspace) return hipErrorInvalidValue;
        kv8_index_kernel<<<dim3((unsigned)((a.num_tokens + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream>>>(
            a.slot_mapping, (int)a.num_tokens, a.num_cache_blocks * a.block_size, a.workspace);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    if (fast_shape(dt, a))
        return fmt == Kv8Format::Int8 ? launch_fast<Kv8Format::Int8>(a, indexed, stream)
                                      : launch_fast<Kv8Format::E4M3>(a, indexed, stream);
    if (dt == DType::BF16)
        return fmt == Kv8Format::Int8 ? launch_generic<__bf16, Kv8Format::Int8>(a, indexed, stream)
                                      : launch_generic<__bf16, Kv8Format::E4M3>(a, indexed, stream);
    return fmt == Kv8Format::Int8 ? launch_generic<float, Kv8Format::Int8>(a, indexed, stream)
                                  : launch_generic<float, Kv8Format::E4M3>(a, indexed, stream);
}

hipError_t launch_kv8_gather(DType dt, Kv8Format fmt, const void *k_cache, const void *v_cache,
                             const float *k_scales, const float *v_scales, const int32_t *ids, int64_t num_ids,
                             void *k_out, void *v_out, int64_t num_cache_blocks, int block_size, int num_kv_heads,
                             int head_dim, hipStream_t stream) {
    if (num_ids <= 0) return hipSuccess;
    const auto at = [](const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    const bool wide = head_dim % 8 == 0 && at(k_cache, 8) && at(v_cache, 8) && at(k_out, 16) && at(v_out, 16);
#define NVLLM_KV8_GATHER(ET, F)                                                                                  \
    return wide ? launch_gather<ET, F, 8>(k_cache, v_cache, k_scales, v_scales, ids, num_ids, k_out, v_out,      \
                                          num_cache_blocks, block_size, num_kv_heads, head_dim, stream)          \
                : launch_gather<ET, F, 1>(k_cache, v_cache, k_scales, v_scales, ids, num_ids, k_out, v_out,      \
                                          num_cache_blocks, block_size, num_kv_heads, head_dim, stream)
    if (dt == DType::BF16) {
        if (fmt == Kv8Format::Int8) NVLLM_KV8_GATHER(__bf16, Kv8Format::Int8);
        NVLLM_KV8_GATHER(__bf16, Kv8Format::E4M3);
    }
    if (fmt == Kv8Format::Int8) NVLLM_KV8_GATHER(float, Kv8Format::Int8);
    NVLLM_KV8_GATHER(float, Kv8Format::E4M3);
#undef NVLLM_KV8_GATHER
}

}  // namespace kernels
}  // namespace nvllm

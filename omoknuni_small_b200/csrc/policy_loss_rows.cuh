// The kernels of the policy losses (policy_loss.cu), one translation unit per type of logits.
//
// With M the largest legal logit, d_j = z_j - M, e_j = exp(d_j), s = sum e, t = sum e d, p_j = e_j / s, both gradients need
// no more than sums over the row:
//   H(p) = log s - t / s                                 dH/dz_j  = -p_j (d_j - t / s)
//   KL(p|q) = a / s - log s + log b                      dKL/dz_j = p_j (d_j - d'_j - a / s)
//     with d', b those of q's logits and a = sum e (d - d')
//   cross entropy = log s - a / b,  a = sum target d, b = sum target
//                                                        d/dz_j   = p_j - target_j / b
//   clipped term: d/dz_j = k ([j = action] - p_j),  k = -advantage r or 0
// so a gradient is p_j (k0 + kz d_j + kd (d_j - d'_j)) plus a term of the action or of the target.
//
// Rows are worked on in shared memory, where bulk copies bring them while an SM's other teams work on theirs: once for
// the maximum (where actions that do not count are replaced by a lowest value, so that the other passes ask no mask), once
// for the sums, once for the gradient, which leaves in 16-byte stores.  Every matrix is read from memory once and the
// gradient written once.  Instructions matter next to memory: at 6.5 TB/s an SM has 33 thread instructions for an action of
// 16-bit logits with a reference row (6 bytes), 66 in fp32.  Hence the packed arithmetic (two fp32 an instruction), the
// packed 16-bit maximum, and few threads a row, each with many actions.  No unit is full, though (1,024 x 32,768 bf16 with a
// reference: memory 34 %, issue slots 50 %, powers of two 46 %): a row's copy, maximum, sums and gradient come one after the
// other, and shared memory holds the rows of 20 to 24 warps an SM.
//   policy_warp_rows_kernel   short rows: 8, 16 or 32 lanes a row, so that what a row costs besides its actions is paid
//                             once for up to four of them
//   policy_cta_rows_kernel    the others: a CTA or the CTAs of a cluster a row
//   policy_long_rows_kernel   rows beyond the shared memory of eight CTAs, three times through device memory
#pragma once
#include "common.h"
#include "internal.h"
#include "packed_f32.cuh"
#include "sm100_ptx.cuh"
#include <atomic>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace ob200 {

enum PolicyKind { kSearch = 0, kClipped = 1, kClippedRef = 2 };

struct PolicyRows {
    const void* z; const void* x;       // logits; target or reference logits
    const uint32_t* bits; const float* weight;
    void* grad; float* loss; float4* stats;
    long long z_pitch, x_pitch, g_pitch;
    int n, A, mask_words;
    int phase;                          // element of its 16 bytes at which row 0 starts, the same in all three matrices; -1: not the same
    int visits;                         // search: the target is int32
    const int32_t* action; const float* old_logp; const float* advantage;
    float entropy, kl, lo, hi;
};

int launch_policy_rows_f32(int kind, const PolicyRows& r, cudaStream_t st);
int launch_policy_rows_bf16(int kind, const PolicyRows& r, cudaStream_t st);
int launch_policy_rows_f16(int kind, const PolicyRows& r, cudaStream_t st);
uint32_t policy_spin_limit();           // polls before a wait for a row gives up (policy_loss.cu)

#ifdef __CUDACC__
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_inff();
// Differences below it count as it, so that products with a probability of 0 are 0.
template <typename T> constexpr float kLow = -1e30f;
template <> constexpr float kLow<__nv_bfloat16> = -0x1.92p99f;   // the value of bf16 next to it, which stands for it in a row (Lowest)

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN when either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float warp_max_nan(float v) {
    float y;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xFFFFFFFF;" : "=f"(y) : "f"(v));
    return y;
}
// Over the LANES lanes of a team.
template <int LANES = 32>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}
// Four sums over the warp in 6 exchanges instead of 20: lane i ends with the sum of the (i mod 4)th.
__device__ __forceinline__ float four_sums(float s, float t, float a, float b) {
    const int lane = threadIdx.x % 32;
    const bool odd = lane & 1, high = lane & 2;
    const float u = (odd ? t : s) + __shfl_xor_sync(~0u, odd ? s : t, 1), v = (odd ? b : a) + __shfl_xor_sync(~0u, odd ? a : b, 1);
    float w = (high ? v : u) + __shfl_xor_sync(~0u, high ? u : v, 2);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) w += __shfl_xor_sync(~0u, w, o);
    return w;
}
template <int LANES = 32>
__device__ __forceinline__ float team_max_nan(float v) {
    if (LANES == 32) return warp_max_nan(v);
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

__device__ __forceinline__ f32x2 ex2_2(f32x2 v) {
    float a, b;
    halves(v, a, b);
    return pair(ex2(a), ex2(b));
}
// ---- 16 bytes of a row ------------------------------------------------------------
// The value that stands for logits that do not count, and for those below it: in every element of a word, and as fp32.
// A row whose largest logit is below half of it is worked on separately (careful_row).
// fp16 has no value so low that it could stand for a legal -inf: those stay, and threads that met one work with the passes
// that look for them (FLOOR).
template <typename T> struct Lowest;
template <> struct Lowest<float> { static constexpr uint32_t kWord = 0xF149F2CAu; static constexpr float kValue = kLow<float>; };
template <> struct Lowest<__nv_bfloat16> { static constexpr uint32_t kWord = 0xF149F149u; static constexpr float kValue = kLow<__nv_bfloat16>; };
template <> struct Lowest<__half> { static constexpr uint32_t kWord = 0xFBFFFBFFu; static constexpr float kValue = -65504.f; };

// Elements 2i and 2i + 1 of a vector of T as fp32.
template <typename T>
__device__ __forceinline__ f32x2 elements(const uint32_t* v, int i) {
    if (sizeof(T) == 4) return pair(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
    if (std::is_same<T, __nv_bfloat16>::value) return pair(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xFFFF0000u));
    const float2 f = __half22float2(*(const __half2*)&v[i]);
    return pair(f.x, f.y);
}
// The same less c (given as -c), in fp32: a 16-bit operand needs no conversion of its own.
template <typename T, bool FLOOR = false>
__device__ __forceinline__ f32x2 elements_less(const uint32_t* v, int i, f32x2 minus_c, float c) {
    if (sizeof(T) == 4) return add2(elements<T>(v, i), minus_c);
    float a, b;
    if (std::is_same<T, __nv_bfloat16>::value)
        asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; sub.rn.f32.bf16 %0, l, %3; sub.rn.f32.bf16 %1, h, %3;}" : "=f"(a), "=f"(b) : "r"(v[i]), "f"(c));
    else
        asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; sub.rn.f32.f16 %0, l, %3; sub.rn.f32.f16 %1, h, %3;}" : "=f"(a), "=f"(b) : "r"(v[i]), "f"(c));
    if (FLOOR) { a = max_nan(a, kLow<T>); b = max_nan(b, kLow<T>); }
    return pair(a, b);
}
// The larger values of two words, element by element, NaN where either is.
template <typename T>
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b) {
    uint32_t y;
    if (sizeof(T) == 4) asm("max.NaN.f32 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    else if (std::is_same<T, __nv_bfloat16>::value) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
// Whether a word of fp16, the smallest elements met, has a -inf.
template <typename T>
__device__ __forceinline__ bool has_minus_inf(uint32_t low) {
    return std::is_same<T, __half>::value && ((low & 0xFFFFu) == 0xFC00u || low >> 16 == 0xFC00u);
}
template <typename T>
__device__ __forceinline__ float word_top(uint32_t w) {
    if (sizeof(T) == 4) return __uint_as_float(w);
    const uint32_t v[1] = {w};
    float a, b;
    halves(elements<T>(v, 0), a, b);
    return max_nan(a, b);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *(const uint32_t*)&v;
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *(const uint32_t*)&v;
}
// Masks of the eight 16-bit elements of a vector whose bits in `on` are set, word by word.
__device__ __forceinline__ void word_masks(uint32_t on, uint32_t (&m)[4]) {
    // four bits to the signs of four bytes, each sign over a half word
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t signs = ((on >> (4 * i)) & 15u) * 0x10204080u;
        asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m[2 * i]) : "r"(signs));
        asm("prmt.b32 %0, %1, 0, 0xBBAA;" : "=r"(m[2 * i + 1]) : "r"(signs));
    }
}
// 16 bytes and words of shared memory, by their 32-bit address.
__device__ __forceinline__ void load16(uint32_t at, uint32_t* to) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(to[0]), "=r"(to[1]), "=r"(to[2]), "=r"(to[3]) : "r"(at));
}
__device__ __forceinline__ void store16(uint32_t at, const uint32_t* v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ uint32_t load_word(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
template <typename T> __device__ __forceinline__ T* in_shared(uint32_t at) { return (T*)__cvta_shared_to_generic(at); }

// ---- what a row comes to --------------------------------------------------------------
// Sums of a part of a row, relative to its largest logit m and largest reference logit c.
struct Sums { float m, c, s, t, a, b, za; };     // za: the action's logit, -inf when it is not in this part or not legal

// gradient = p (k0 + kz d + kd (d - d')) + ka [action] - kt target,  p = 2^(d log2 e + lp)
struct RowGrad { float M, C, lp, k0, kz, kd, ka, kt; };
struct RowOut { float loss; float4 stats; };

// False when the row is left out.
template <int KIND>
__device__ __forceinline__ bool row_result(const PolicyRows& r, const Sums& q, float w, float old_logp, float adv, RowGrad* g, RowOut* o) {
    const float l2s = lg2(q.s), ls = l2s * kLn2, inv_s = __fdividef(1.f, q.s), mean = q.t * inv_s, H = ls - mean;
    g->M = q.m; g->C = q.c; g->lp = -l2s;
    g->kz = w * r.entropy; g->kd = 0.f; g->ka = 0.f; g->kt = 0.f;
    if (KIND == kSearch) {
        const float inv_T = __fdividef(1.f, q.b), ce = fmaf(-q.a, inv_T, ls);
        g->k0 = w * (1.f - r.entropy * mean);
        g->kt = w * inv_T;
        o->loss = w * (ce - r.entropy * H);
        o->stats = make_float4(ce, H, q.b, q.m + ls);
        return q.b != 0.f;
    }
    const float logp = (q.za - q.m) - ls;
    const float ratio = ex2((logp - old_logp) * kLog2e);
    const float open = ratio * adv, held = fminf(fmaxf(ratio, r.lo), r.hi) * adv;
    const bool free = open <= held || open != open, none = adv == 0.f;
    const float surrogate = none ? 0.f : free ? open : held, k = none || !free ? 0.f : -open;
    float kl = 0.f, ud = 0.f;
    g->kd = w * r.kl;
    if (KIND == kClippedRef) {
        ud = q.a * inv_s;
        kl = ud - (l2s - lg2(q.b)) * kLn2;
        if (kl != kl) ud = kl;
        // The reference gives no legal action any probability: KL is infinite whatever p is, and has no gradient.
        if (q.b == 0.f) { kl = kInf; ud = g->kd = 0.f; }
    }
    g->k0 = w * (-k - r.kl * ud - r.entropy * mean);
    g->ka = w * k;
    o->loss = w * (-surrogate + (r.kl == 0.f && kl == kInf ? 0.f : r.kl * kl) - r.entropy * H);
    o->stats = make_float4(logp, ratio, kl, H);
    return q.za != -kInf;
}

__device__ __forceinline__ void put_out(const PolicyRows& r, long long row, bool live, const RowOut& o) {
    if (r.loss) r.loss[row] = live ? o.loss : 0.f;
    if (r.stats) r.stats[row] = live ? o.stats : make_float4(0.f, 0.f, 0.f, 0.f);
}

// Targets whose sum T, times differences down to -1e30 and as a divisor of a row's weight, stays well within fp32: a row with
// others is scaled by a power of two, by careful_row.  NaN is taken as it is.
__device__ __forceinline__ bool target_fits(float T) { return !(T > 0x1p27f || (T < 0x1p-60f && T != 0.f)); }
// Largest logits beyond the floor's size: differences from them would be below it where the other passes do not look.
template <typename T> __device__ __forceinline__ bool too_high(float m) { return !std::is_same<T, __half>::value && m > -kLow<T>; }

__device__ __forceinline__ bool legal(const uint32_t* bits, int j) { return !bits || (bits[j >> 5] >> (j & 31)) & 1u; }
__device__ __forceinline__ float target_f32(uint32_t raw, int visits) { return visits ? (float)(int)raw : __uint_as_float(raw); }

// ---- a row straight from device memory ---------------------------------------------------
// `threads` threads (a warp, or a CTA of 512) go over a row three times; join(v, is_max) joins a value over them.
template <typename T, int KIND, typename Join>
__device__ __forceinline__ void plain_row(const PolicyRows& r, long long row, int tid, int threads, Join join) {
    const T* z = (const T*)r.z + row * r.z_pitch;
    const uint8_t* x = (const uint8_t*)r.x + row * r.x_pitch * (KIND == kSearch ? 4 : sizeof(T));
    T* grad = (T*)r.grad + row * r.g_pitch;
    const uint32_t* bits = r.bits ? r.bits + row * r.mask_words : nullptr;
    const float w = r.weight ? r.weight[row] : 1.f;
    const int act = KIND == kSearch ? -1 : r.action[row];
    auto second = [&](int j) { return KIND == kSearch ? target_f32(((const uint32_t*)x)[j], r.visits) : KIND == kClippedRef ? to_f32(((const T*)x)[j]) : 0.f; };
    Sums q{-kInf, -kInf, 0.f, 0.f, 0.f, 0.f, -kInf};
    bool live = w != 0.f;
    if (live && bits) {
        float some = 0.f;
        for (int i = tid; i < (r.A + 31) / 32; i += threads)
            if (bits[i] & (i == r.A / 32 ? ~(~0u << (r.A & 31)) : ~0u)) some = 1.f;
        live = join(some, true) != 0.f;
    }
    if (live)
#pragma unroll 4
        for (int j = tid; j < r.A; j += threads)
            if (legal(bits, j)) {
                const float v = to_f32(z[j]);
                q.m = max_nan(q.m, v);
                if (KIND == kClippedRef) q.c = max_nan(q.c, second(j));
                if (KIND != kSearch && j == act) q.za = v == -kInf ? -3.4e38f : v;
            }
    q.m = join(q.m, true);
    if (KIND == kClippedRef) q.c = join(q.c, true);
    if (KIND != kSearch) q.za = join(q.za, true);
    live = live && q.m != -kInf;
    if (KIND != kClippedRef || q.c == -kInf) q.c = 0.f;
    if (live)
#pragma unroll 4
        for (int j = tid; j < r.A; j += threads)
            if (legal(bits, j)) {
                const float d = to_f32(z[j]) - q.m, e = ex2(d * kLog2e), dl = fmaxf(d, kLow<T>), y = second(j);
                q.s += e;
                q.t = fmaf(e, dl, q.t);
                if (KIND == kSearch) { q.a = fmaf(y, dl, q.a); q.b += y; }
                if (KIND == kClippedRef) { q.a = fmaf(e, dl - fmaxf(y - q.c, kLow<T>), q.a); q.b += ex2((y - q.c) * kLog2e); }
            }
    q.s = join(q.s, false); q.t = join(q.t, false);
    if (KIND != kClipped) { q.a = join(q.a, false); q.b = join(q.b, false); }
    const float total = q.b;
    float unit = 1.f;                            // of the targets
    if (KIND == kSearch && !target_fits(total)) {
        unit = __uint_as_float((254u - min(max((__float_as_uint(total) & 0x7FFFFFFFu) >> 23, 1u), 253u)) << 23);
        q.a = q.b = 0.f;
        if (live)
            for (int j = tid; j < r.A; j += threads)
                if (legal(bits, j)) {
                    const float y = second(j) * unit;
                    q.a = fmaf(y, fmaxf(to_f32(z[j]) - q.m, kLow<T>), q.a);
                    q.b += y;
                }
        q.a = join(q.a, false); q.b = join(q.b, false);
    }
    if (q.za != -kInf) q.za = max_nan(q.za, q.m + kLow<T>);
    RowGrad g;
    RowOut out;
    live = row_result<KIND>(r, q, w, KIND == kSearch ? 0.f : r.old_logp[row], KIND == kSearch ? 0.f : r.advantage[row], &g, &out) && live;
    if (KIND == kSearch) out.stats.z = total;
    if (tid == 0) put_out(r, row, live, out);
#pragma unroll 4
    for (int j = tid; j < r.A; j += threads) {
        float o = 0.f;
        if (live && legal(bits, j)) {
            const float d = to_f32(z[j]) - g.M, dl = fmaxf(d, kLow<T>), y = second(j);
            o = fmaf(g.kz, dl, g.k0);
            if (KIND == kClippedRef) o = fmaf(g.kd, dl - fmaxf(y - g.C, kLow<T>), o);
            o *= ex2(fmaf(d, kLog2e, g.lp));
            if (KIND == kSearch) o = fmaf(-g.kt, y * unit, o);
            else if (j == act) o += g.ka;
        }
        grad[j] = from_f32<T>(o);
    }
}

// Rows without an ordinary logit (all of them at a type's lowest value or -inf), with one beyond 1e30 or with targets of
// an extreme scale, by one warp.
template <typename T, int KIND>
__device__ __noinline__ void careful_row(const PolicyRows& r, long long row) {
    plain_row<T, KIND>(r, row, threadIdx.x % 32, 32, [](float v, bool is_max) { return is_max ? warp_max_nan(v) : team_sum(v); });
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A cluster of eight CTAs a row: 148 rows of 400,000 fp32 actions with a reference 499 us, one row 76 (a CTA a row: 1,397 and 510).
constexpr int kLongCtas = 8;
template <typename T, int KIND>
__global__ void __cluster_dims__(kLongCtas) __launch_bounds__(512)
policy_long_rows_kernel(const __grid_constant__ PolicyRows r) {
    __shared__ float part[2][kLongCtas * 16];
    uint32_t cta;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int turn = 0;
    cluster_barrier();                           // the others write into this CTA's shared memory
    plain_row<T, KIND>(r, blockIdx.x / kLongCtas, (int)cta * 512 + threadIdx.x, kLongCtas * 512, [&](float v, bool is_max) {
        v = is_max ? warp_max_nan(v) : team_sum(v);
        if (lane < kLongCtas) {
            uint32_t there;
            asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(ptx::smem_u32(&part[turn][cta * 16 + warp])), "r"(lane));
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(v) : "memory");
        }
        cluster_barrier();
        const float *p = part[turn] + lane, a = p[0], b = p[32], c = p[64], d = p[96];
        turn ^= 1;
        return is_max ? warp_max_nan(max_nan(max_nan(a, b), max_nan(c, d))) : team_sum((a + b) + (c + d));
    });
    cluster_barrier();
}

// ---- rows in shared memory ------------------------------------------------------------
// How rows lie there.  A slot holds a CTA's or warp team's part of a row: a header, vectors of 16 bytes of logits, what
// belongs to them of the second matrix, and the words of the mask.
struct RowShape {
    int seg;                            // vectors a CTA holds of a row
    int x_at, mask_at, slot_bytes;      // offsets in a slot, its size
    uint32_t spins;
    int* error;
};
constexpr int kHeader = 32;             // weight, old log-probability, advantage, action; head, vectors, -, flags

__device__ __forceinline__ void copy_word_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void arrive_after_copies(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
}


// Where a row lies within its vectors: the first element's place, vectors; whether the outer vectors reach beyond the
// matrices (else their ends hold what stands beside the row, which the first pass replaces).
struct Place { int head, vecs; bool first_out, last_out; };
template <typename T, int KIND, bool ALIKE>
__device__ __forceinline__ Place place_of(const PolicyRows& r, long long row) {
    constexpr int V = 16 / sizeof(T), XB = KIND == kSearch ? 4 : (int)sizeof(T);
    Place p{0, (r.A + V - 1) / V, false, false};
    if (ALIKE) {
        p.head = (r.phase + (int)(row & (V - 1)) * (int)(r.z_pitch & (V - 1))) & (V - 1);
        p.vecs = (p.head + r.A + V - 1) / V;
        // only the rows at the ends of a matrix can reach beyond it, and with rows shorter than a vector their neighbours
        if (row < V || row >= r.n - V) {
            const long long lo = row * r.z_pitch - p.head, xlo = row * r.x_pitch - p.head, end = (long long)p.vecs * V;
            p.first_out = lo < 0 || (KIND != kClipped && xlo < 0);
            p.last_out = lo + end > (r.n - 1) * r.z_pitch + r.A || (KIND != kClipped && xlo + end > (r.n - 1) * r.x_pitch + r.A);
        }
    }
    return p;
}

// A team's part of a row in its slot.
struct Part {
    uint32_t zs, xs, ms;                // addresses in shared memory; ms: words of the mask from mask_first on
    int mask_first, head, vecs, v0, v1; // this part's vectors are [v0, v1)
    bool first_out, last_out;
};

// What the first pass finds in its vectors: the largest words of both matrices; fp16: the smallest of either.
struct Tops { uint32_t z, x, low; };
__device__ __forceinline__ void word_min(uint32_t& low, uint32_t w) { asm("min.f16x2 %0, %0, %1;" : "+r"(low) : "r"(w)); }

// The words of vector v of a part.
template <typename T, int KIND>
struct Vec {
    static constexpr int V = 16 / sizeof(T), XB = KIND == kSearch ? 4 : (int)sizeof(T), XW = KIND == kClipped ? 1 : V * XB / 4;
    uint32_t z[4], x[XW];
    __device__ __forceinline__ void load_z(const Part& p, int v) { load16(p.zs + (v - p.v0) * 16, z); }
    __device__ __forceinline__ void load_x(const Part& p, int v) {
        if (KIND != kClipped)
#pragma unroll
            for (int i = 0; i < XW / 4; ++i) load16(p.xs + (v - p.v0) * (XW * 4) + 16 * i, x + 4 * i);
    }
    __device__ __forceinline__ void store_z(const Part& p, int v) const { store16(p.zs + (v - p.v0) * 16, z); }
    __device__ __forceinline__ void store_x(const Part& p, int v) const {
        if (KIND != kClipped)
#pragma unroll
            for (int i = 0; i < XW / 4; ++i) store16(p.xs + (v - p.v0) * (XW * 4) + 16 * i, x + 4 * i);
    }
    // Elements without their bit in `on` become the lowest value, their targets 0.
    __device__ __forceinline__ void keep(uint32_t on) {
        if (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool is = on & (1u << i);
                z[i] = is ? z[i] : Lowest<T>::kWord;
                if (KIND == kClippedRef) x[i % XW] = is ? x[i % XW] : Lowest<T>::kWord;
                if (KIND == kSearch) x[i % XW] = is ? x[i % XW] : 0u;
            }
        } else {
            uint32_t m[4];
            word_masks(on, m);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                z[i] = (z[i] & m[i]) | (Lowest<T>::kWord & ~m[i]);
                if (KIND == kClippedRef) x[i % XW] = (x[i % XW] & m[i]) | (Lowest<T>::kWord & ~m[i]);
            }
            if (KIND == kSearch)
#pragma unroll
                for (int i = 0; i < V; ++i) x[i % XW] = on & (1u << i) ? x[i % XW] : 0u;
        }
    }
    __device__ __forceinline__ void counts_to_f32() {
#pragma unroll
        for (int i = 0; i < XW; ++i) x[i] = __float_as_uint((float)(int)x[i]);
    }
    // The largest words; not below the lowest value, or, in fp16, the smallest words too.
    __device__ __forceinline__ void raise(Tops& t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (std::is_same<T, __half>::value) word_min(t.low, z[i]);
            else z[i] = word_max<T>(z[i], Lowest<T>::kWord);
            t.z = word_max<T>(t.z, z[i]);
            if (KIND == kClippedRef) {
                if (std::is_same<T, __half>::value) word_min(t.low, x[i % XW]);
                else x[i % XW] = word_max<T>(x[i % XW], Lowest<T>::kWord);
                t.x = word_max<T>(t.x, x[i % XW]);
            }
        }
    }
};

// Vectors of a part that lie in the row as a whole: [lo, hi); the outer ones, or -1.
struct Inner { int lo, hi, first, last; };
template <int V>
__device__ __forceinline__ Inner inner_of(const PolicyRows& r, const Part& p) {
    const bool head = p.head != 0, tail = ((p.head + r.A) & (V - 1)) != 0;
    Inner n{p.v0, p.v1, -1, -1};
    if (head && p.v0 == 0 && p.v1 > 0) { n.first = 0; n.lo = 1; }
    if (tail && p.v1 == p.vecs && p.v1 > n.lo) { n.last = p.vecs - 1; n.hi = p.v1 - 1; }
    return n;
}

// Bits of the legal actions of vector v; the places ahead of the row and behind it have none (the word ahead of the mask's
// first is 0, what stands behind its last is cut off).
template <int V>
__device__ __forceinline__ uint32_t bits_of(const PolicyRows& r, const Part& p, int v) {
    const int j = v * V - p.head;                           // the first element's action; below 0 in the first vector
    uint32_t on = ~0u;
    if (r.bits) {
        const uint32_t w = p.ms + 4 * ((j >> 5) - p.mask_first);
        on = __funnelshift_r(load_word(w), load_word(w + 4), j & 31);
    } else if (j < 0) {
        on <<= -j;
    }
    if (j + V > r.A) on &= ~(~0u << (r.A - j));
    return on;
}

// An outer vector that was not copied, because it reaches beyond the matrix, element by element.
template <typename T, int KIND>
__device__ __noinline__ void fetch_vector(const PolicyRows& r, long long row, const Part& p, int v) {
    constexpr int V = 16 / sizeof(T);
    const int j = v * V - p.head, at = (v - p.v0) * V;
    for (int i = 0; i < V; ++i)
        if (j + i >= 0 && j + i < r.A) {
            in_shared<T>(p.zs)[at + i] = ((const T*)r.z)[row * r.z_pitch + j + i];
            if (KIND == kSearch) in_shared<uint32_t>(p.xs)[at + i] = ((const uint32_t*)r.x)[row * r.x_pitch + j + i];
            if (KIND == kClippedRef) in_shared<T>(p.xs)[at + i] = ((const T*)r.x)[row * r.x_pitch + j + i];
        }
}

// First pass, over vectors v0 + tid, + stride ...: the largest words; what does not count becomes the lowest value (a target
// 0), visit counts become fp32.  Returns whether any action met was legal.
// SHORT: rows of a few vectors a thread take their outer vectors along in the loop; the others' loops are free of them.
template <typename T, int KIND, bool ALIKE, int U, bool SHORT>
__device__ __forceinline__ bool pass_max(const PolicyRows& r, long long row, const Part& p, int tid, int stride, Tops& tops) {
    constexpr int V = 16 / sizeof(T);
    uint32_t any = r.bits ? 0u : ~0u;
    using W = Vec<T, KIND>;
    const Inner n = inner_of<V>(r, p);
    int v = p.v0 + tid;
    if (SHORT) {
        if (ALIKE && (p.first_out || p.last_out)) {
            if (p.first_out && tid == 0 && p.v1 > 0) fetch_vector<T, KIND>(r, row, p, 0);
            if (p.last_out && p.v1 > 0 && (p.vecs - 1) % stride == tid) fetch_vector<T, KIND>(r, row, p, p.vecs - 1);
        }
        for (; v < p.v1; v += stride) {
            W w;
            w.load_z(p, v);
            const bool edge = v == n.first || v == n.last, change = r.bits || edge;
            if (KIND == kClippedRef || (KIND == kSearch && (change || r.visits))) w.load_x(p, v);
            if (change) {
                const uint32_t on = bits_of<V>(r, p, v);
                any |= on & ((1u << V) - 1);
                w.keep(on);
            }
            if (KIND == kSearch && r.visits) w.counts_to_f32();
            w.raise(tops);
            w.store_z(p, v);
            if (KIND == kClippedRef || (KIND == kSearch && (change || r.visits))) w.store_x(p, v);
        }
        return any != 0u;
    }
    if (v < n.lo) v += stride;
    if (r.bits) {
        for (; v < n.hi; v += stride) {
            W w;
            w.load_z(p, v);
            w.load_x(p, v);
            const int j = v * V - p.head;
            const uint32_t bits = p.ms + 4 * ((j >> 5) - p.mask_first);
            const uint32_t on = __funnelshift_r(load_word(bits), load_word(bits + 4), j & 31);
            any |= on & ((1u << V) - 1);
            w.keep(on);
            if (KIND == kSearch) {
                if (r.visits) w.counts_to_f32();
                w.store_x(p, v);
            }
            w.raise(tops);
            w.store_z(p, v);
            if (KIND == kClippedRef) w.store_x(p, v);
        }
    } else if (KIND == kSearch && r.visits) {
        for (; v < n.hi; v += stride) {
            W w;
            w.load_z(p, v);
            w.load_x(p, v);
            w.counts_to_f32();
            w.store_x(p, v);
            w.raise(tops);
            w.store_z(p, v);
        }
    } else {
        for (; v + (U - 1) * stride < n.hi; v += U * stride) {
            W w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                w[u].load_z(p, v + u * stride);
                if (KIND == kClippedRef) w[u].load_x(p, v + u * stride);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                w[u].raise(tops);
                w[u].store_z(p, v + u * stride);
                if (KIND == kClippedRef) w[u].store_x(p, v + u * stride);
            }
        }
        for (; v < n.hi; v += stride) {
            W w;
            w.load_z(p, v);
            if (KIND == kClippedRef) w.load_x(p, v);
            w.raise(tops);
            w.store_z(p, v);
            if (KIND == kClippedRef) w.store_x(p, v);
        }
    }
    for (int k = 0; k < 2; ++k) {
        // the first vector is thread 0's; the last one's thread has come to it by its steps
        const int e = k ? n.last : n.first;
        if (e < 0 || (k ? v != e : tid != 0)) continue;
        if (ALIKE && ((e == 0 && p.first_out) || (e == p.vecs - 1 && p.last_out))) fetch_vector<T, KIND>(r, row, p, e);
        W w;
        w.load_z(p, e);
        w.load_x(p, e);
        const uint32_t on = bits_of<V>(r, p, e);
        any |= on & ((1u << V) - 1);
        w.keep(on);
        if (KIND == kSearch && r.visits) w.counts_to_f32();
        w.raise(tops);
        w.store_z(p, e);
        w.store_x(p, e);
    }
    return any != 0u;
}

// Second pass: the sums relative to q.m and q.c.
template <typename T, int KIND, int U, bool FLOOR>
__device__ __forceinline__ void pass_sums(const Part& p, int tid, int stride, Sums& q) {
    constexpr int V = 16 / sizeof(T);
    using W = Vec<T, KIND>;
    const f32x2 M = pair(-q.m, -q.m), C = pair(-q.c, -q.c), L = pair(kLog2e, kLog2e), minus = pair(-1.f, -1.f);
    f32x2 s = 0, t = 0, a = 0, b = 0;
    auto add = [&](const W& w) {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const f32x2 d = elements_less<T, FLOOR>(w.z, i, M, q.m), e = ex2_2(mul2(d, L));
            s = add2(s, e);
            t = fma2(e, d, t);
            if (KIND == kSearch) {
                const f32x2 y = elements<float>(w.x, i);
                a = fma2(y, d, a);
                b = add2(b, y);
            }
            if (KIND == kClippedRef) {
                const f32x2 c = elements_less<T, FLOOR>(w.x, i, C, q.c);
                b = add2(b, ex2_2(mul2(c, L)));
                a = fma2(e, fma2(c, minus, d), a);
            }
        }
    };
    int v = p.v0 + tid;
    for (; v + (U - 1) * stride < p.v1; v += U * stride) {
        W w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) { w[u].load_z(p, v + u * stride); w[u].load_x(p, v + u * stride); }
#pragma unroll
        for (int u = 0; u < U; ++u) add(w[u]);
    }
    for (; v < p.v1; v += stride) {
        W w;
        w.load_z(p, v);
        w.load_x(p, v);
        add(w);
    }
    q.s = sum2(s); q.t = sum2(t); q.a = sum2(a); q.b = sum2(b);
}

// Third pass: the gradient (0 where the row is not live), to `grad` (the row's element 0 stands at grad + head), or into
// the slot where stores of vectors are not possible.
template <typename T, int KIND, bool ALIKE, int U, bool SHORT, bool FLOOR>
__device__ __forceinline__ void pass_grad(const PolicyRows& r, const Part& p, int tid, int stride, bool live, const RowGrad& g, int act_e, T* grad) {
    constexpr int V = 16 / sizeof(T);
    using W = Vec<T, KIND>;
    const f32x2 M = pair(-g.M, -g.M), C = pair(-g.C, -g.C), L = pair(kLog2e, kLog2e);
    // kz d + kd (d - d') as (kz + kd) d - kd d'
    const float kzd = g.kz + g.kd;
    const f32x2 lp = pair(g.lp, g.lp), k0 = pair(g.k0, g.k0), kz = pair(kzd, kzd), kd = pair(-g.kd, -g.kd), kt = pair(-g.kt, -g.kt);
    const Inner n = ALIKE ? inner_of<V>(r, p) : Inner{p.v0, p.v1, -1, -1};
    // The action's element has a term of its own: its thread makes it apart and stores it over the vector's, so that the
    // loops ask nothing of it.
    const int act_at = act_e - p.v0 * V;
    const bool act_mine = KIND != kSearch && live && act_e >= p.v0 * V && act_e < p.v1 * V && act_at / V % stride == tid;
    float act_grad = 0.f;
    if (act_mine) {
        const float d = max_nan(to_f32(in_shared<const T>(p.zs)[act_at]) - g.M, kLow<T>);
        float y = fmaf(kzd, d, g.k0);
        if (KIND == kClippedRef) y = fmaf(-g.kd, max_nan(to_f32(in_shared<const T>(p.xs)[act_at]) - g.C, kLow<T>), y);
        act_grad = fmaf(y, ex2(fmaf(d, kLog2e, g.lp)), g.ka);
    }
    auto put_act = [&] {
        if (!act_mine) return;
        if (ALIKE) grad[act_e] = from_f32<T>(act_grad);
        else in_shared<T>(p.zs)[act_at] = from_f32<T>(act_grad);
    };
    // the gradient's words in place of the logits'
    auto made = [&](W& w) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const f32x2 d = elements_less<T, FLOOR>(w.z, i, M, g.M), pr = ex2_2(fma2(d, L, lp));
            f32x2 y = fma2(kz, d, k0);
            if (KIND == kClippedRef) y = fma2(kd, elements_less<T, FLOOR>(w.x, i, C, g.C), y);
            y = mul2(y, pr);
            if (KIND == kSearch) y = fma2(kt, elements<float>(w.x, i), y);
            halves(y, o[2 * i], o[2 * i + 1]);
        }
        if (sizeof(T) == 4)
#pragma unroll
            for (int i = 0; i < 4; ++i) w.z[i] = __float_as_uint(o[i % V]);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) w.z[i] = pack2<T>(o[(2 * i) % V], o[(2 * i + 1) % V]);
    };
    auto put = [&](const W& w, int v) {
        if (ALIKE) *(uint4*)(grad + v * V) = make_uint4(w.z[0], w.z[1], w.z[2], w.z[3]);
        else w.store_z(p, v);
    };
    int v = p.v0 + tid;
    if (SHORT && ALIKE) {
        const int end = p.head + r.A;
#pragma unroll 2
        for (; v < p.v1; v += stride) {
            W w;
            w.z[0] = w.z[1] = w.z[2] = w.z[3] = 0u;
            if (live) {
                w.load_z(p, v);
                w.load_x(p, v);
                made(w);
            }
            if (v != n.first && v != n.last) {
                put(w, v);
            } else {
                const int at = v * V;
                T* to = grad + at;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const uint32_t word = w.z[i * (int)sizeof(T) / 4];
                    if (at + i >= p.head && at + i < end) {
                        if (sizeof(T) == 4) *(uint32_t*)(to + i) = word;
                        else *(unsigned short*)(to + i) = (unsigned short)(i & 1 ? word >> 16 : word);
                    }
                }
            }
        }
        put_act();
        return;
    }
    if (v < n.lo) v += stride;
    if (live) {
        for (; v + (U - 1) * stride < n.hi; v += U * stride) {
            W w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) { w[u].load_z(p, v + u * stride); w[u].load_x(p, v + u * stride); }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                made(w[u]);
                put(w[u], v + u * stride);
            }
        }
        for (; v < n.hi; v += stride) {
            W w;
            w.load_z(p, v);
            w.load_x(p, v);
            made(w);
            put(w, v);
        }
    } else {
        W w;
        w.z[0] = w.z[1] = w.z[2] = w.z[3] = 0u;
        for (; v < n.hi; v += stride) put(w, v);
    }
    if (!ALIKE) {
        put_act();
        return;
    }
    for (int k = 0; k < 2; ++k) {
        const int e = k ? n.last : n.first;
        if (e < 0 || (k ? v != e : tid != 0)) continue;
        W w;
        w.z[0] = w.z[1] = w.z[2] = w.z[3] = 0u;
        if (live) {
            w.load_z(p, e);
            w.load_x(p, e);
            made(w);
        }
        w.store_z(p, e);
        const int at = e * V;
        for (int i = max(p.head - at, 0); i < min(V, p.head + r.A - at); ++i) grad[at + i] = in_shared<const T>(p.zs)[(e - p.v0) * V + i];
    }
    put_act();
}

// The action's logit from element `at` of the slot; -inf as a difference of it counts.
template <typename T>
__device__ __forceinline__ float action_logit(const Part& p, int at) { return max_nan(to_f32(in_shared<const T>(p.zs)[at]), kLow<T>); }

// Without vectors: what a team holds of a row, element by element, into its slot and back.
template <typename T, int KIND>
__device__ __forceinline__ void copy_in(const PolicyRows& r, long long row, const Part& p, int tid, int stride) {
    constexpr int V = 16 / sizeof(T);
    const int j0 = p.v0 * V, j1 = min(p.v1 * V, r.A);
    for (int j = j0 + tid; j < j1; j += stride) {
        in_shared<T>(p.zs)[j - j0] = ((const T*)r.z)[row * r.z_pitch + j];
        if (KIND == kSearch) in_shared<uint32_t>(p.xs)[j - j0] = ((const uint32_t*)r.x)[row * r.x_pitch + j];
        if (KIND == kClippedRef) in_shared<T>(p.xs)[j - j0] = ((const T*)r.x)[row * r.x_pitch + j];
    }
    if (r.bits)
        for (int i = p.mask_first + tid; i <= (j1 - 1) >> 5; i += stride) in_shared<uint32_t>(p.ms)[i - p.mask_first] = r.bits[row * r.mask_words + i];
}
template <typename T>
__device__ __forceinline__ void copy_out(const PolicyRows& r, const Part& p, int tid, int stride, T* grad) {
    constexpr int V = 16 / sizeof(T);
    const int j0 = p.v0 * V, j1 = min(p.v1 * V, r.A);
    for (int j = j0 + tid; j < j1; j += stride) grad[j] = in_shared<const T>(p.zs)[j - j0];
}

__device__ __forceinline__ float4 scalars_of(const PolicyRows& r, int kind, long long row) {
    float4 v = make_float4(1.f, 0.f, 0.f, 0.f);
    if (row >= r.n) return v;
    if (r.weight) v.x = r.weight[row];
    if (kind != kSearch) { v.y = r.old_logp[row]; v.z = r.advantage[row]; v.w = __int_as_float(r.action[row]); }
    return v;
}

// The copies of vectors [v0, v1) of a row into a slot, announced at and counted by bar.
template <typename T, int KIND>
__device__ __forceinline__ void copy_vectors(const PolicyRows& r, long long row, const Place& p, int v0, int v1, uint32_t slot, int x_at, uint32_t bar, bool wanted) {
    constexpr int V = 16 / sizeof(T), XB = KIND == kSearch ? 4 : (int)sizeof(T), XV = V * XB;
    int lo = v0, hi = v1;
    if (lo == 0 && p.first_out) lo = 1;
    if (hi == p.vecs && p.last_out) --hi;
    const int n = hi - lo;
    if (!wanted || n <= 0) {
        ptx::mbar_arrive(bar);
        return;
    }
    ptx::mbar_arrive_expect_tx(bar, n * (KIND == kClipped ? 16 : 16 + XV));
    const uint8_t* z = (const uint8_t*)r.z + (row * r.z_pitch - p.head + (long long)lo * V) * (int)sizeof(T);
    ptx::bulk_g2s(slot + kHeader + (lo - v0) * 16, z, n * 16, bar);
    if (KIND != kClipped) {
        const uint8_t* x = (const uint8_t*)r.x + (row * r.x_pitch - p.head + (long long)lo * V) * XB;
        ptx::bulk_g2s(slot + x_at + (lo - v0) * XV, x, n * XV, bar);
    }
}

// What a team whose copy did not arrive leaves of its rows from `row` on: NaN, so that no update is made of them (rows of
// weight 0 as ever).
template <typename T>
__device__ __noinline__ void lost_rows(const PolicyRows& r, long long row, long long step, int tid, int threads) {
    for (; row < r.n; row += step) {
        const float y = r.weight && r.weight[row] == 0.f ? 0.f : __int_as_float(0x7fc00000);
        if (tid == 0) put_out(r, row, true, RowOut{y, make_float4(y, y, y, y)});
        for (int j = tid; j < r.A; j += threads) ((T*)r.grad)[row * r.g_pitch + j] = from_f32<T>(y);
    }
}

// ---- short rows --------------------------------------------------------------------
// LANES lanes a row, 32 / LANES adjacent rows a warp; each warp has slots of its own and fills them itself.  While a warp waits
// for its copies the SM's others work: with two slots a warp, and so half the warps, 65,536 x 362 took 90 us, with one 52.
template <typename T, int KIND, int LANES, bool ALIKE>
__global__ void __launch_bounds__(128, LANES == 32 ? 4 : 6)
policy_warp_rows_kernel(const __grid_constant__ PolicyRows r, const __grid_constant__ RowShape sh) {
    constexpr int R = 32 / LANES, U = LANES == 32 ? 4 : 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int abort_flag;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32, tid = lane % LANES, mine_of = lane / LANES;
    const int warp_bytes = R * sh.slot_bytes + 16;
    uint8_t* const mine = smem + warp * warp_bytes;
    const uint32_t mine_s = ptx::smem_u32(mine), full = mine_s + R * sh.slot_bytes;
    if (ALIKE && lane == 0) ptx::mbar_init(full, R + (r.bits ? 32 : 0));
    if (threadIdx.x == 0) abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();

    const long long first = ((long long)blockIdx.x * warps + warp) * R + mine_of, step = (long long)gridDim.x * warps * R;
    uint8_t* const at = mine + mine_of * sh.slot_bytes;
    const uint32_t at_s = mine_s + mine_of * sh.slot_bytes;
    // This team's row into its slot; rows beyond the last are announced too, so that the warp's barrier completes.
    auto fill = [&](long long row, float4 scalars) {
        const bool is = row < r.n;
        if (r.bits) {
            if (is)
                for (int i = tid; i < (r.A + 31) / 32; i += LANES) copy_word_async(at_s + sh.mask_at + 4 * i, r.bits + row * r.mask_words + i);
            arrive_after_copies(full);
        }
        if (tid == 0) {
            *(float4*)at = scalars;
            const Place p = place_of<T, KIND, ALIKE>(r, is ? row : 0);
            copy_vectors<T, KIND>(r, row, p, 0, p.vecs, at_s, sh.x_at, full, is && scalars.x != 0.f);
        }
    };
    if (r.bits && tid == 0) *(uint32_t*)(at + sh.mask_at - 4) = 0u;
    __syncwarp();
    float4 ahead = make_float4(0.f, 0.f, 0.f, 0.f);          // scalars of the row after the one in the slot
    if (ALIKE) {
        if (first - mine_of < r.n) fill(first, scalars_of(r, KIND, first));
        if (tid == 0) ahead = scalars_of(r, KIND, first + step);
    }
    uint32_t parity = 0;
    for (long long row = first; row - mine_of < r.n; row += step) {        // the same turns for the whole warp
        const bool is = row < r.n;
        const Place pl = place_of<T, KIND, ALIKE>(r, is ? row : 0);
        const Part p{at_s + kHeader, at_s + sh.x_at, at_s + sh.mask_at, 0, pl.head, pl.vecs, 0, is ? pl.vecs : 0, pl.first_out, pl.last_out};
        float4 scalars;
        if (ALIKE) {
            if (!ptx::mbar_wait_warp(full, parity, &abort_flag, sh.spins)) {
                abort_flag = 1;
                atomicExch(sh.error, 4);
                int none = 0;
                ptx::mbar_wait(full, parity, &none);             // what is in flight is waited for once more
                lost_rows<T>(r, row, step, tid, LANES);
                break;
            }
            parity ^= 1;
            scalars = *(const float4*)at;
        } else {
            scalars = scalars_of(r, KIND, row);
            if (is && scalars.x != 0.f) copy_in<T, KIND>(r, row, p, tid, LANES);
            __syncwarp();
        }
        const float w = scalars.x;
        const int act = KIND == kSearch ? -1 : __float_as_int(scalars.w);
        const int act_e = (unsigned)act < (unsigned)r.A ? act + p.head : -1;       // the action's element of the row
        bool live = is && w != 0.f, apart = false;
        Tops tops{Lowest<T>::kWord, Lowest<T>::kWord, Lowest<T>::kWord};
        const bool some = live && pass_max<T, KIND, ALIKE, U, (LANES < 32)>(r, row, p, tid, LANES, tops);
        const bool floored = std::is_same<T, __half>::value && __any_sync(~0u, has_minus_inf<T>(tops.low));
        // rows without a legal action are left out
        if (LANES == 32) live = __any_sync(~0u, some);
        else live = (__ballot_sync(~0u, some) >> (lane & ~(LANES - 1))) & ((1u << (LANES & 31)) - 1);
        Sums q;
        q.m = team_max_nan<LANES>(word_top<T>(tops.z));
        q.c = KIND == kClippedRef ? team_max_nan<LANES>(word_top<T>(tops.x)) : 0.f;
        __syncwarp();
        q.za = -kInf;
        if (KIND != kSearch && live && act_e >= 0 && (!r.bits || (load_word(p.ms + 4 * (act >> 5)) >> (act & 31)) & 1u)) q.za = action_logit<T>(p, act_e);
        apart = live && (q.m < Lowest<T>::kValue / 2 || too_high<T>(q.m) || (KIND == kClippedRef && (q.c < Lowest<T>::kValue / 2 || too_high<T>(q.c))));
        q.s = q.t = q.a = q.b = 0.f;
        if (live && !apart) {
            if (floored) pass_sums<T, KIND, U, true>(p, tid, LANES, q);
            else pass_sums<T, KIND, U, false>(p, tid, LANES, q);
        }
        q.s = team_sum<LANES>(q.s);
        q.t = team_sum<LANES>(q.t);
        if (KIND != kClipped) { q.a = team_sum<LANES>(q.a); q.b = team_sum<LANES>(q.b); }
        if (KIND == kSearch && live && !target_fits(q.b)) apart = true;
        live = live && !apart;
        RowGrad g;
        RowOut out;
        live = row_result<KIND>(r, q, w, scalars.y, scalars.z, &g, &out) && live;
        if (tid == 0 && is && !apart) put_out(r, row, live, out);
        T* const grad = (T*)r.grad + row * r.g_pitch - p.head;
        __syncwarp();                            // the gradient may take the place of the action's logit
        if (!apart) {
            if (floored) pass_grad<T, KIND, ALIKE, U, (LANES < 32), true>(r, p, tid, LANES, live, g, act_e, grad);
            else pass_grad<T, KIND, ALIKE, U, (LANES < 32), false>(r, p, tid, LANES, live, g, act_e, grad);
        }
        for (uint32_t m = __ballot_sync(~0u, apart && tid == 0); m; m &= m - 1)
            careful_row<T, KIND>(r, __shfl_sync(~0u, row, __ffs(m) - 1));
        if (ALIKE) {
            // the slot's next copy comes behind what was read and written here
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (row - mine_of + step < r.n) {
                fill(row + step, ahead);
                if (tid == 0) ahead = scalars_of(r, KIND, row + 2 * step);
            }
        } else {
            __syncwarp();
            if (!apart) copy_out<T>(r, p, tid, LANES, grad);
            __syncwarp();
        }
    }
}

// ---- rows of a CTA or a cluster ----------------------------------------------------------
// What a warp or a CTA found of a row, relative to its own largest logit m and reference logit c - or to 0 where it has no
// ordinary one: its terms are 0 then.
template <typename T>
__device__ __forceinline__ float base_of(float top) { return top < Lowest<T>::kValue / 2 ? 0.f : top; }
// Entries (m, c, s, t | a, b, za, whether any action is legal), one a lane, none in lanes from n on, as one.
template <typename T, int KIND>
__device__ __forceinline__ Sums join_entries(const float (*entry)[8], int n) {
    const int lane = threadIdx.x % 32;
    const float* mine = entry[lane < n ? lane : 0];
    const float4 lo = *(const float4*)mine, hi = *(const float4*)(mine + 4);
    Sums q;
    q.m = warp_max_nan(lo.x);
    q.c = KIND == kClippedRef ? warp_max_nan(lo.y) : 0.f;
    q.za = KIND == kSearch ? 0.f : warp_max_nan(hi.z);
    q.s = q.t = q.a = q.b = 0.f;
    if (lane < n) {
        const float d = base_of<T>(lo.x) - base_of<T>(q.m), f = lo.z == 0.f ? 0.f : ex2(d * kLog2e);
        q.s = lo.z * f;
        q.t = fmaf(d, q.s, lo.w * f);
        if (KIND == kSearch) { q.a = fmaf(d, hi.y, hi.x); q.b = hi.y; }
        if (KIND == kClippedRef) {
            const float dc = base_of<T>(lo.y) - base_of<T>(q.c);
            q.a = fmaf(d - dc, q.s, hi.x * f);
            q.b = hi.y == 0.f ? 0.f : hi.y * ex2(dc * kLog2e);
        }
    }
    const float sum = four_sums(q.s, q.t, q.a, q.b);
    q.s = __shfl_sync(~0u, sum, 0); q.t = __shfl_sync(~0u, sum, 1); q.a = __shfl_sync(~0u, sum, 2); q.b = __shfl_sync(~0u, sum, 3);
    return q;
}

// A CTA, or a cluster's CTAs, a row.  A warp's sums are relative to its own maxima and are joined by every warp at once, so
// that a row costs one meeting of its warps, and one more before its slot takes the next row; while a CTA waits for its
// copy the SM's others work.
// (A run of the row for each warp to itself, copied in one, two or four pieces that refill as soon as their gradient has left,
// and no second meeting: 4,096 x 32,768 bf16 199, 213, 225 us against 196, 2,048 x 4,672 25, 27, 29 against 21; what it costs
// in instructions is more than the waits that it saves.)
template <typename T, int KIND, bool ALIKE>
__global__ void __launch_bounds__(256, 3)
policy_cta_rows_kernel(const __grid_constant__ PolicyRows r, const __grid_constant__ RowShape sh) {
    constexpr int V = 16 / sizeof(T), U = 2;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(16) float part[2][32][8];        // the sums of the cluster's warps, by turns
    __shared__ __align__(8) unsigned long long full_bar;
    __shared__ int abort_flag;
    uint32_t cta, ctas;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, threads = blockDim.x, warps = threads / 32;
    const uint32_t smem_s = ptx::smem_u32(smem), full = ptx::smem_u32(&full_bar);
    if (threadIdx.x == 0) {
        ptx::mbar_init(full, 1 + (r.bits ? 32 : 0));
        if (r.bits) *(uint32_t*)(smem + sh.mask_at - 4) = 0u;
        abort_flag = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    // the cluster's CTAs write into each other's shared memory: all of them have to be there
    if (ctas > 1) cluster_barrier();
    const int v0 = (int)cta * sh.seg;
    const long long first = blockIdx.x / ctas, step = gridDim.x / ctas;
    // A row into the slot, by the first warp.
    auto fill = [&](long long row, float4 scalars) {
        const Place p = place_of<T, KIND, ALIKE>(r, row);
        const int v1 = min(p.vecs, v0 + sh.seg);
        if (r.bits) {
            const int w0 = max(v0 * V - p.head, 0) >> 5, w1 = (min(v1 * V - p.head, r.A) - 1) >> 5;
            for (int i = w0 + lane; i <= w1; i += 32) copy_word_async(smem_s + sh.mask_at + 4 * (i - w0), r.bits + row * r.mask_words + i);
            arrive_after_copies(full);
        }
        if (lane == 0) {
            *(float4*)smem = scalars;
            *(int4*)(smem + 16) = make_int4(p.head, p.vecs, 0, (p.first_out ? 1 : 0) | (p.last_out ? 2 : 0));
            copy_vectors<T, KIND>(r, row, p, v0, v1, smem_s, sh.x_at, full, scalars.x != 0.f);
        }
    };
    float4 ahead;                                // scalars of the row after the one in the slot
    if (ALIKE && warp == 0) {
        if (first < r.n) fill(first, scalars_of(r, KIND, first));
        ahead = scalars_of(r, KIND, first + step);
    }
    uint32_t parity = 0, filled = 0;             // of the row's barrier phase; of the last row filled
    int turn = 0;
    for (long long row = first; row < r.n; row += step) {
        float4 scalars;
        Place pl;
        // The row's copy did not arrive, or an earlier one's: no slot is filled any more.  Its scalars, which all warps of a
        // row have to agree on, come from where the slot has them from, and its sums are NaN.
        bool lost = false;
        if (ALIKE) {
            lost = __any_sync(~0u, *(volatile int*)&abort_flag);
            if (!lost && !ptx::mbar_wait_warp(full, parity, &abort_flag, sh.spins)) {
                lost = true;
                abort_flag = 1;
                atomicExch(sh.error, 4);
            }
            parity ^= 1;
        }
        if (ALIKE && !lost) {
            scalars = *(const float4*)smem;
            const int4 h = *(const int4*)(smem + 16);
            pl = Place{h.x, h.y, (h.w & 1) != 0, (h.w & 2) != 0};
        } else {
            scalars = scalars_of(r, KIND, row);
            pl = place_of<T, KIND, ALIKE>(r, row);
        }
        const Part p{smem_s + kHeader, smem_s + sh.x_at, smem_s + sh.mask_at, max(v0 * V - pl.head, 0) >> 5, pl.head, pl.vecs,
                     v0, min(pl.vecs, v0 + sh.seg), pl.first_out, pl.last_out};
        const float w = scalars.x;
        if (!ALIKE) {
            if (w != 0.f) copy_in<T, KIND>(r, row, p, threadIdx.x, threads);
            __syncthreads();
        }
        const int act = KIND == kSearch ? -1 : __float_as_int(scalars.w);
        const int act_e = (unsigned)act < (unsigned)r.A ? act + p.head : -1;       // the action's element of the row
        bool live = w != 0.f, apart = false, floored = false;
        RowGrad g;
        RowOut out;
        if (live) {                              // the same in the whole team
            Tops tops{Lowest<T>::kWord, Lowest<T>::kWord, Lowest<T>::kWord};
            const bool some = __any_sync(~0u, pass_max<T, KIND, ALIKE, U, false>(r, row, p, threadIdx.x, threads, tops)) || lost;
            floored = std::is_same<T, __half>::value && __any_sync(~0u, has_minus_inf<T>(tops.low));
            float top = warp_max_nan(word_top<T>(tops.z)), top_ref = KIND == kClippedRef ? warp_max_nan(word_top<T>(tops.x)) : 0.f;
            __syncwarp();
            // The action's logit, by the warp that has its vector and ahead of the meeting: behind it the others may find the
            // gradient in its place.
            const int act_at = KIND != kSearch && act_e >= v0 * V && act_e < p.v1 * V && (!r.bits || (load_word(p.ms + 4 * ((act >> 5) - p.mask_first)) >> (act & 31)) & 1u)
                                   ? act_e - v0 * V : -1;
            float za = -kInf;
            if (KIND != kSearch && act_at >= 0 && act_at / V % threads / 32 == warp) za = action_logit<T>(p, act_at);
            Sums q;
            q.m = base_of<T>(top);
            q.c = KIND == kClippedRef ? base_of<T>(top_ref) : 0.f;
            if (floored) pass_sums<T, KIND, U, true>(p, threadIdx.x, threads, q);
            else pass_sums<T, KIND, U, false>(p, threadIdx.x, threads, q);
            float sum = four_sums(q.s, q.t, q.a, q.b);
            if (lost) top = top_ref = sum = za = __int_as_float(0x7fc00000);
            float (*all)[8] = part[turn];
            turn ^= 1;
            float* const mine = all[cta * warps + warp];
            if (ctas == 1) {
                if (lane < 4) mine[2 + lane] = sum;
                else if (lane == 4) { mine[0] = top; mine[1] = top_ref; mine[6] = za; mine[7] = some ? 1.f : 0.f; }
                __syncthreads();
            } else {
                const float s = __shfl_sync(~0u, sum, 0), t = __shfl_sync(~0u, sum, 1), a = __shfl_sync(~0u, sum, 2), b = __shfl_sync(~0u, sum, 3);
                if (lane < (int)ctas) {
                    uint32_t there;
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(ptx::smem_u32(mine)), "r"(lane));
                    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there), "f"(top), "f"(top_ref), "f"(s), "f"(t) : "memory");
                    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there + 16), "f"(a), "f"(b), "f"(za), "f"(some ? 1.f : 0.f) : "memory");
                }
                cluster_barrier();
            }
            q = join_entries<T, KIND>(all, (int)ctas * warps);
            const bool legal_one = __any_sync(~0u, lane < (int)ctas * warps && all[lane][7] != 0.f);      // else the row is left out
            apart = legal_one && (q.m < Lowest<T>::kValue / 2 || too_high<T>(q.m) || (KIND == kSearch && !target_fits(q.b)) ||
                                  (KIND == kClippedRef && (q.c < Lowest<T>::kValue / 2 || too_high<T>(q.c))));
            live = row_result<KIND>(r, q, w, scalars.y, scalars.z, &g, &out) && legal_one;
            if (apart && warp == 0 && cta == 0) careful_row<T, KIND>(r, row);
        }
        if (threadIdx.x == 0 && cta == 0 && !apart) put_out(r, row, live, out);
        T* const grad = (T*)r.grad + row * r.g_pitch - p.head;
        if (!apart) {
            if (floored) pass_grad<T, KIND, ALIKE, U, false, true>(r, p, threadIdx.x, threads, live, g, act_e, grad);
            else pass_grad<T, KIND, ALIKE, U, false, false>(r, p, threadIdx.x, threads, live, g, act_e, grad);
        }
        if (ALIKE) {
            // the next copy comes behind what was read and written here
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncthreads();
            if (warp == 0 && row + step < r.n && !*(volatile int*)&abort_flag) {
                filled ^= 1;
                fill(row + step, ahead);
                ahead = scalars_of(r, KIND, row + 2 * step);
            }
        } else {
            __syncthreads();
            if (!apart) copy_out<T>(r, p, threadIdx.x, threads, grad);
            __syncthreads();
        }
    }
    if (ALIKE && abort_flag && threadIdx.x == 0) {       // what is still in flight is waited for once more
        int none = 0;
        ptx::mbar_wait(full, filled, &none);
    }
    __syncthreads();
    // and none may leave while another may still write
    if (ctas > 1) cluster_barrier();
}

// ---- host ---------------------------------------------------------------------------
constexpr int kSms = 148;
constexpr int kMostShared = 208 * 1024;          // of a CTA; 227 KB less the kernels' own

// Registers of a thread | SMs << 16.  Looked up once for each kernel and device, where the kernel is also given its shared
// memory.
struct KernelFacts { std::atomic<int> of[64]; };
template <typename Kernel>
int kernel_facts(Kernel kernel, KernelFacts* known, int* facts, int* device = nullptr) {
    int dev = 0, sms = 0;
    OB200_CUDA_OK(cudaGetDevice(&dev));
    if (device) *device = dev;
    if (dev < 64 && (*facts = known->of[dev].load(std::memory_order_acquire)) != 0) return OB200_OK;
    cudaFuncAttributes a;
    OB200_CUDA_OK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    OB200_CUDA_OK(cudaFuncGetAttributes(&a, kernel));
    OB200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
    *facts = a.numRegs | sms << 16;
    if (dev < 64) known->of[dev].store(*facts, std::memory_order_release);
    return OB200_OK;
}
// CTAs the device holds at once.
int resident_ctas(int facts, int threads, int smem) {
    const int by_regs = 65536 / (((facts & 0xFFFF) + 7) / 8 * 8 * threads), by_smem = 226 * 1024 / (smem + 4 * 1024), by_threads = 2048 / threads;
    int n = by_regs < by_smem ? by_regs : by_smem;
    n = n < by_threads ? n : by_threads;
    return (facts >> 16) * (n < 1 ? 1 : n);
}

template <typename T, int KIND, int LANES, bool ALIKE>
int launch_warp_rows(const PolicyRows& r, const RowShape& sh, cudaStream_t st) {
    constexpr int R = 32 / LANES;
    static KernelFacts known;
    auto kernel = policy_warp_rows_kernel<T, KIND, LANES, ALIKE>;
    int facts;
    if (int rc = kernel_facts(kernel, &known, &facts)) return rc;
    const int warp_bytes = R * sh.slot_bytes + 16, fit = 104 * 1024 / warp_bytes, warps = fit < 1 ? 1 : fit > 4 ? 4 : fit;
    const long long teams = ((long long)r.n + R * warps - 1) / (R * warps), room = resident_ctas(facts, 32 * warps, warps * warp_bytes);
    kernel<<<(unsigned)(teams < room ? teams : room), 32 * warps, warps * warp_bytes, st>>>(r, sh);
    OB200_LAUNCHED("policy_warp_rows_kernel");
    return OB200_OK;
}

template <typename T, int KIND, bool ALIKE>
int launch_cta_rows(const PolicyRows& r, const RowShape& sh, int warps, int ctas, cudaStream_t st) {
    static KernelFacts known;
    auto kernel = policy_cta_rows_kernel<T, KIND, ALIKE>;
    int facts, dev;
    if (int rc = kernel_facts(kernel, &known, &facts, &dev)) return rc;
    const int threads = 32 * warps, smem = sh.slot_bytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)ctas, 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = ctas > 1 ? 1 : 0;
    long long room = resident_ctas(facts, threads, smem);
    if (ctas > 1) {
        // Fewer clusters fit than their CTAs would: not every group of SMs divides into them.  Each cluster has its share of
        // the rows, so one that had to wait for another's end would double the time.  The answer is kept for the next call
        // with the same shape on the same device.
        static std::atomic<uint64_t> last[4];
        std::atomic<uint64_t>& slot = last[ctas == 2 ? 0 : ctas == 4 ? 1 : 2];
        const uint64_t key = (uint64_t)dev << 52 | (uint64_t)smem << 32 | (uint64_t)threads << 16;
        uint64_t got = slot.load(std::memory_order_relaxed);
        if ((got & ~0xFFFFULL) != key) {
            int n = 0;
            OB200_CUDA_OK(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
            got = key | (uint64_t)(n < 1 ? 1 : n);
            slot.store(got, std::memory_order_relaxed);
        }
        room = (long long)(got & 0xFFFF);
    }
    cfg.gridDim = dim3((unsigned)((r.n < room ? r.n : room) * ctas));
    cudaLaunchKernelEx(&cfg, kernel, r, sh);
    OB200_LAUNCHED("policy_cta_rows_kernel");
    return OB200_OK;
}

template <typename T, int KIND, bool ALIKE>
int launch_shape(const PolicyRows& r, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T), XV = KIND == kClipped ? 0 : V * (KIND == kSearch ? 4 : (int)sizeof(T));
    const int vecs = (int)(((long long)r.A + (ALIKE ? V - 1 : 0) + V - 1) / V);
    RowShape sh{};
    sh.error = device_error_word();
    sh.spins = policy_spin_limit();
    if (!sh.error) return set_error(OB200_ERR_CUDA, "policy loss: the device's error word is not available");
    auto lay = [&](int ctas) {
        sh.seg = (vecs + ctas - 1) / ctas;
        sh.x_at = kHeader + sh.seg * 16;
        sh.mask_at = sh.x_at + sh.seg * XV + (r.bits ? 4 : 0);        // behind a word that is 0; a word more than is copied is read
        sh.slot_bytes = (sh.mask_at + (r.bits ? (sh.seg * V / 32 + 3) * 4 : 0) + 15) / 16 * 16;
        return sh.slot_bytes;
    };
    if (r.A <= 1024) {
        lay(1);
        // More rows than the device holds warps for at once: several rows a warp, as far as the shared memory of 24 warps
        // allows (100,000 x 225 fp32: 60 us with 8 lanes a row, 88 with 16, 133 with 32).  Fewer: a warp each (512 x 225: 5.3
        // us, 8 lanes 7.2).
        const bool many = r.n > 24 * kSms;
        if (ALIKE && many && sh.slot_bytes <= 2400) return launch_warp_rows<T, KIND, ALIKE ? 8 : 32, ALIKE>(r, sh, st);
        if (ALIKE && many && sh.slot_bytes <= 4800) return launch_warp_rows<T, KIND, ALIKE ? 16 : 32, ALIKE>(r, sh, st);
        return launch_warp_rows<T, KIND, 32, ALIKE>(r, sh, st);
    }
    if ((long long)vecs * (16 + XV) <= 8LL * kMostShared) {
        // A row's part takes up to a third of an SM's shared memory (4,096 x 32,768 bf16: 193 us in parts of 65 KB, 232 in
        // parts of 33 KB).  While SMs are left over, smaller parts (8 x 32,768: 5.6 us with eight CTAs a row, 8.5 with two).
        int ctas = 1;
        while (ctas < 8 && lay(ctas) > 72 * 1024) ctas *= 2;
        while (ctas < 8 && lay(ctas) > 20 * 1024 && (long long)r.n * ctas < 2 * kSms) ctas *= 2;
        if (lay(ctas) <= kMostShared) {
            // 64 actions a lane, as few as there may be while every row has SMs of its own; 32 entries of sums at most
            const int most = ctas == 8 ? 4 : 8, lanes_of = (long long)r.n * ctas < 2 * kSms ? 16 : 64;
            const int warps = (sh.seg * V + 32 * lanes_of - 1) / (32 * lanes_of);
            return launch_cta_rows<T, KIND, ALIKE>(r, sh, warps > most ? most : warps, ctas, st);
        }
    }
    if ((long long)r.n * kLongCtas > 0x7fffffffLL) return set_error(OB200_ERR_TOO_LARGE, "policy loss: %d rows of %d actions", r.n, r.A);
    policy_long_rows_kernel<T, KIND><<<(unsigned)(r.n * kLongCtas), 512, 0, st>>>(r);
    OB200_LAUNCHED("policy_long_rows_kernel");
    return OB200_OK;
}

template <typename T>
int launch_policy_rows(int kind, const PolicyRows& r, cudaStream_t st) {
    const bool alike = r.phase >= 0;
    if (kind == kSearch) return alike ? launch_shape<T, kSearch, true>(r, st) : launch_shape<T, kSearch, false>(r, st);
    if (kind == kClipped) return alike ? launch_shape<T, kClipped, true>(r, st) : launch_shape<T, kClipped, false>(r, st);
    return alike ? launch_shape<T, kClippedRef, true>(r, st) : launch_shape<T, kClippedRef, false>(r, st);
}

}  // namespace
#endif
}  // namespace ob200

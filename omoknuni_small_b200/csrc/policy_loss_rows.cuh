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
// A team - a warp, a CTA, or the CTAs of a cluster - works on a row that bulk copies have brought into shared memory while
// it was busy with the row before: once for the maximum (where actions that do not count are replaced by -inf, so that the
// other passes ask no mask), once for the sums, once for the gradient, which leaves in 16-byte stores.  Every matrix is
// read from memory once and the gradient written once.  What bounds the kernel next to memory is instructions: at
// 6.5 TB/s an SM has 33 thread instructions for an action of 16-bit logits with a reference row (6 bytes), 66 in fp32;
// hence the packed arithmetic (two fp32 an instruction), the packed 16-bit maximum, and few threads a row, each with many
// actions, over which the joining of sums is spread.
#pragma once
#include "common.h"
#include "internal.h"
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

#ifdef __CUDACC__
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_inff();
constexpr float kLow = -1e30f;          // differences below it count as it, so that products with a probability of 0 are 0

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
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Two fp32 in a register pair.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
    f32x2 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void halves(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ f32x2 ex2_2(f32x2 v) {
    float a, b;
    halves(v, a, b);
    return pair(ex2(a), ex2(b));
}
__device__ __forceinline__ f32x2 floor2(f32x2 v) {            // not below kLow
    float a, b;
    halves(v, a, b);
    return pair(fmaxf(a, kLow), fmaxf(b, kLow));
}
__device__ __forceinline__ float sum2(f32x2 v) {
    float a, b;
    halves(v, a, b);
    return a + b;
}

// ---- 16 bytes of a row ------------------------------------------------------------
template <typename T> struct Bits;                              // per type: -inf in every element of a word
template <> struct Bits<float> { static constexpr uint32_t kNinf = 0xFF800000u; };
template <> struct Bits<__nv_bfloat16> { static constexpr uint32_t kNinf = 0xFF80FF80u; };
template <> struct Bits<__half> { static constexpr uint32_t kNinf = 0xFC00FC00u; };

// Elements 2i and 2i + 1 of a vector of T as fp32.
template <typename T>
__device__ __forceinline__ f32x2 elements(const uint32_t* v, int i) {
    if (sizeof(T) == 4) return pair(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
    if (std::is_same<T, __nv_bfloat16>::value) return pair(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xFFFF0000u));
    const float2 f = __half22float2(*(const __half2*)&v[i]);
    return pair(f.x, f.y);
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
// Masks of the elements of a vector whose bits in `on` are set, word by word.
template <typename T>
__device__ __forceinline__ void word_masks(uint32_t on, uint32_t (&m)[4]) {
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = (on >> i) & 1u ? ~0u : 0u;
    } else {
        // four bits to the signs of four bytes, each sign over a half word
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t signs = ((on >> (4 * i)) & 15u) * 0x10204080u;
            asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m[2 * i]) : "r"(signs));
            asm("prmt.b32 %0, %1, 0, 0xBBAA;" : "=r"(m[2 * i + 1]) : "r"(signs));
        }
    }
}
__device__ __forceinline__ void load16(const uint8_t* p, uint32_t* to) {
    const uint4 v = *(const uint4*)p;
    to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
}
__device__ __forceinline__ void store16(uint8_t* p, const uint32_t* v) { *(uint4*)p = make_uint4(v[0], v[1], v[2], v[3]); }

// ---- what a row comes to --------------------------------------------------------------
// Sums of a part of a row, relative to its largest logit m and largest reference logit c.
struct Sums { float m, c, s, t, a, b, za; };     // za: the action's logit, -inf when it is not in this part or not legal

// gradient = p (k0 + kz d + kd (d - d')) + ka [action] - kt target,  p = 2^(d log2 e + lp)
struct RowGrad { float M, C, lp, k0, kz, kd, ka, kt; };
struct RowOut { float loss; float4 stats; };

// False when the row is left out.
template <int KIND>
__device__ __forceinline__ bool row_result(const PolicyRows& r, const Sums& q, float w, float old_logp, float adv, RowGrad* g, RowOut* o) {
    if (q.m == -kInf) return false;
    const float l2s = lg2(q.s), ls = l2s * kLn2, inv_s = __fdividef(1.f, q.s), mean = q.t * inv_s, H = ls - mean;
    g->M = q.m; g->C = q.c == -kInf ? 0.f : q.c; g->lp = -l2s;
    g->kz = w * r.entropy; g->kd = 0.f; g->ka = 0.f; g->kt = 0.f;
    if (KIND == kSearch) {
        if (!(q.b != 0.f)) return false;
        const float inv_T = 1.f / q.b, ce = fmaf(-q.a, inv_T, ls);
        g->k0 = w * (1.f - r.entropy * mean);
        g->kt = w * inv_T;
        o->loss = w * (ce - r.entropy * H);
        o->stats = make_float4(ce, H, q.b, q.m + ls);
        return true;
    }
    if (q.za == -kInf) return false;
    const float logp = max_nan(q.za - q.m, kLow) - ls;
    const float ratio = ex2((logp - old_logp) * kLog2e);
    float surrogate = 0.f, k = 0.f;
    if (adv != 0.f) {
        const float open = ratio * adv, held = fminf(fmaxf(ratio, r.lo), r.hi) * adv;
        surrogate = open <= held ? open : held;
        k = open <= held ? -open : 0.f;
        if (open != open) surrogate = k = open;
    }
    float kl = 0.f, ud = 0.f;
    if (KIND == kClippedRef) {
        ud = q.a * inv_s;
        kl = q.b == 0.f ? kInf : ud - (l2s - lg2(q.b)) * kLn2;       // 0: q gives nothing to any legal action
        if (kl != kl) ud = kl;
    }
    g->k0 = w * (-k - r.kl * ud - r.entropy * mean);
    g->kd = w * r.kl;
    g->ka = w * k;
    o->loss = w * (-surrogate + r.kl * kl - r.entropy * H);
    o->stats = make_float4(logp, ratio, kl, H);
    return true;
}

__device__ __forceinline__ bool legal(const uint32_t* bits, int j) { return !bits || (bits[j >> 5] >> (j & 31)) & 1u; }
__device__ __forceinline__ float target_f32(uint32_t raw, int visits) { return visits ? (float)(int)raw : __uint_as_float(raw); }

// ---- rows in shared memory ------------------------------------------------------------
// How rows lie there.  A slot holds a team's part of a row: its scalars (16 bytes), vectors of 16 bytes of logits, what
// belongs to them of the second matrix, and the words of the mask.
struct RowShape {
    int seg;                            // vectors a CTA holds of a row
    int x_at, mask_at, slot_bytes;      // offsets in a slot, its size
    int slots, team_bytes;              // slots in turn; bytes of a team's slots and barriers
    int* error;
};

__device__ __forceinline__ void copy_word_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void arrive_after_copies(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
}

// WARP: a warp per row.  Else the CTA, or the cluster's CTAs, work on a row together.  ALIKE: the rows of the matrices start
// at the same element of 16 bytes, so vectors are copied and stored whole; else element by element.
template <typename T, int KIND, bool WARP, bool ALIKE>
__global__ void __launch_bounds__(WARP ? 256 : 512, 2)
policy_rows_kernel(const __grid_constant__ PolicyRows r, const __grid_constant__ RowShape sh) {
    constexpr int V = 16 / sizeof(T), XB = KIND == kSearch ? 4 : (int)sizeof(T), XV = V * XB;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float top_of[2][16][2];
    __shared__ float part[2][128][8];            // what the warps of the team found, by turns
    __shared__ int abort_flag;
    uint32_t cta = 0, ctas = 1;
    if (!WARP) {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    }
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
    const int tid = WARP ? lane : threadIdx.x, team = WARP ? 32 : blockDim.x;
    const long long first = WARP ? (long long)blockIdx.x * warps + warp : blockIdx.x / ctas;
    const long long step = WARP ? (long long)gridDim.x * warps : gridDim.x / ctas;
    uint8_t* const mine = smem + (WARP ? warp * sh.team_bytes : 0);
    const uint32_t mine_s = ptx::smem_u32(mine), bars = mine_s + sh.slots * sh.slot_bytes;
    if (ALIKE && tid == 0)
        for (int s = 0; s < sh.slots; ++s) ptx::mbar_init(bars + 8 * s, r.bits ? 1 + team : 1);
    if (threadIdx.x == 0) abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    // the cluster's CTAs write into each other's shared memory: all of them have to be there
    if (!WARP && ctas > 1) cluster_barrier();

    const int v0 = (int)cta * sh.seg;
    const uintptr_t z0 = (uintptr_t)r.z, x0 = (uintptr_t)r.x;
    const uintptr_t z1 = z0 + ((r.n - 1) * r.z_pitch + r.A) * sizeof(T), x1 = x0 + ((r.n - 1) * r.x_pitch + r.A) * XB;
    // Where row q lies: its first element's place in the first vector, vectors, this CTA's; whether the outer vectors
    // reach beyond the matrices (the others' ends hold what stands beside the row, which the first pass replaces).
    struct Place { int head, vecs, v1; bool first_out, last_out; };
    auto place_of = [&](long long q) {
        Place p;
        p.head = ALIKE ? (int)((r.phase + q * r.z_pitch) % V) : 0;
        p.vecs = (p.head + r.A + V - 1) / V;
        p.v1 = min(p.vecs, v0 + sh.seg);
        const uintptr_t za = z0 + (q * r.z_pitch - p.head) * sizeof(T), xa = x0 + (q * r.x_pitch - p.head) * XB;
        p.first_out = za < z0 || (KIND != kClipped && xa < x0);
        p.last_out = za + p.vecs * 16 > z1 || (KIND != kClipped && xa + (uintptr_t)p.vecs * XV > x1);
        return p;
    };
    // Row q into slot s, asynchronously.  scalars: thread 0's.
    auto fill = [&](long long q, int s, float4 scalars) {
        const uint32_t slot = mine_s + s * sh.slot_bytes, bar = bars + 8 * s;
        const Place p = place_of(q);
        if (r.bits) {
            const int w0 = max(v0 * V - p.head, 0) >> 5, w1 = (min(p.v1 * V - p.head, r.A) - 1) >> 5;
            const uint32_t* from = r.bits + q * r.mask_words;
            for (int i = w0 + tid; i <= w1; i += team) copy_word_async(slot + sh.mask_at + 4 * (i - w0), from + i);
            arrive_after_copies(bar);
        }
        if (tid == 0) {
            *(float4*)(mine + s * sh.slot_bytes) = scalars;
            int lo = v0, hi = p.v1;
            if (lo == 0 && p.first_out) lo = 1;
            if (hi == p.vecs && p.last_out) --hi;
            if (scalars.x != 0.f && hi > lo) {
                const int n = hi - lo;
                const uintptr_t za = z0 + (q * r.z_pitch - p.head) * sizeof(T), xa = x0 + (q * r.x_pitch - p.head) * XB;
                ptx::mbar_arrive_expect_tx(bar, n * (KIND == kClipped ? 16 : 16 + XV));
                ptx::bulk_g2s(slot + 16 + (lo - v0) * 16, (const void*)(za + (uintptr_t)lo * 16), n * 16, bar);
                if (KIND != kClipped) ptx::bulk_g2s(slot + sh.x_at + (lo - v0) * XV, (const void*)(xa + (uintptr_t)lo * XV), n * XV, bar);
            } else {
                ptx::mbar_arrive(bar);
            }
        }
    };
    auto scalars_of = [&](long long q) {
        float4 v = make_float4(1.f, 0.f, 0.f, 0.f);
        if (q >= r.n) return v;
        if (r.weight) v.x = r.weight[q];
        if (KIND != kSearch) { v.y = r.old_logp[q]; v.z = r.advantage[q]; v.w = __int_as_float(r.action[q]); }
        return v;
    };
    float4 ahead = make_float4(0.f, 0.f, 0.f, 0.f);      // scalars of the next row to be copied
    if (ALIKE) {
        for (int s = 0; s < sh.slots; ++s)
            if (first + s * step < r.n) fill(first + s * step, s, scalars_of(first + s * step));
        if (tid == 0) ahead = scalars_of(first + sh.slots * step);
    }

    int slot = 0, turn = 0, part_turn = 0, last_slot = -1;
    uint32_t parity = 0;
    for (long long row = first; row < r.n; row += step) {
        uint8_t* const at = mine + slot * sh.slot_bytes;
        uint8_t *const zs = at + 16, *const xs = at + sh.x_at;
        const uint32_t* const ms = (const uint32_t*)(at + sh.mask_at);
        const Place p = place_of(row);
        const int mask_first = max(v0 * V - p.head, 0) >> 5;
        float4 scalars;
        if (ALIKE) {
            if (!ptx::mbar_wait(bars + 8 * slot, parity, &abort_flag)) { abort_flag = 1; atomicExch(sh.error, 4); }
            scalars = *(const float4*)at;
        } else {
            scalars = scalars_of(row);
            if (scalars.x != 0.f) {
                const int j1 = min(p.v1 * V, r.A);
                const T* z = (const T*)r.z + row * r.z_pitch;
                for (int j = v0 * V + tid; j < j1; j += team) {
                    ((T*)zs)[j - v0 * V] = z[j];
                    if (KIND == kSearch) ((uint32_t*)xs)[j - v0 * V] = ((const uint32_t*)r.x)[row * r.x_pitch + j];
                    if (KIND == kClippedRef) ((T*)xs)[j - v0 * V] = ((const T*)r.x)[row * r.x_pitch + j];
                }
                if (r.bits)
                    for (int i = mask_first + tid; i <= (j1 - 1) >> 5; i += team) ((uint32_t*)ms)[i - mask_first] = r.bits[row * r.mask_words + i];
            }
            if (WARP) __syncwarp(); else __syncthreads();
        }
        const float w = scalars.x;
        const int act = KIND == kSearch ? -1 : __float_as_int(scalars.w);
        const int act_e = (unsigned)act < (unsigned)r.A ? act + p.head : -1;     // the action's element of the row
        bool live = w != 0.f;
        RowGrad g;
        RowOut out{0.f, make_float4(0.f, 0.f, 0.f, 0.f)};

        // the maximum; what does not count becomes -inf (a target 0), visit counts become fp32
        uint32_t top_z = Bits<T>::kNinf, top_x = Bits<T>::kNinf;
        if (live) {
            const int edge_first = p.head ? 0 : -1, edge_last = (p.head + r.A) % V ? p.vecs - 1 : -1;
            for (int v = v0 + tid; v < p.v1; v += team) {
                uint8_t *zp = zs + (v - v0) * 16, *xp = xs + (v - v0) * XV;
                uint32_t z[4], x[XV / 4];
                load16(zp, z);
                const bool edge = v == edge_first || v == edge_last;
                if (KIND == kClippedRef || (KIND == kSearch && (r.bits || r.visits || edge)))
#pragma unroll
                    for (int i = 0; i < XV / 16; ++i) load16(xp + 16 * i, x + 4 * i);
                if (r.bits || edge) {
                    const int j = v * V - p.head;                   // the first element's action; below 0 in the first vector
                    uint32_t on = ~0u;
                    if (r.bits) {
                        const int i = (j >> 5) - mask_first, most = (r.A - 1) >> 5;
                        const uint32_t lo = j < 0 ? 0u : ms[i], hi = (j & 31) + V > 32 && (j >> 5) < most ? ms[i + 1] : 0u;
                        on = __funnelshift_r(lo, hi, j & 31);
                    }
                    if (j < 0) on &= ~0u << -j;
                    if (j + V > r.A) on &= ~(~0u << (r.A - j));
                    if (ALIKE && ((v == 0 && p.first_out) || (v == p.vecs - 1 && p.last_out))) {
                        // not copied: it reaches beyond the matrix
                        for (int i = 0; i < V; ++i)
                            if (j + i >= 0 && j + i < r.A) {
                                ((T*)zp)[i] = ((const T*)r.z)[row * r.z_pitch + j + i];
                                if (KIND == kSearch) ((uint32_t*)xp)[i] = ((const uint32_t*)r.x)[row * r.x_pitch + j + i];
                                if (KIND == kClippedRef) ((T*)xp)[i] = ((const T*)r.x)[row * r.x_pitch + j + i];
                            }
                        load16(zp, z);
                        if (KIND != kClipped)
#pragma unroll
                            for (int i = 0; i < XV / 16; ++i) load16(xp + 16 * i, x + 4 * i);
                    }
                    uint32_t m[4];
                    word_masks<T>(on, m);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        z[i] = (z[i] & m[i]) | (Bits<T>::kNinf & ~m[i]);
                        if (KIND == kClippedRef) x[i] = (x[i] & m[i]) | (Bits<T>::kNinf & ~m[i]);
                    }
                    store16(zp, z);
                    if (KIND == kClippedRef) store16(xp, x);
                    if (KIND == kSearch)
#pragma unroll
                        for (int i = 0; i < V; ++i) x[i] = (on >> i) & 1u ? x[i] : 0u;
                }
                if (KIND == kSearch && (r.bits || r.visits || edge)) {
                    if (r.visits)
#pragma unroll
                        for (int i = 0; i < V; ++i) x[i] = __float_as_uint((float)(int)x[i]);
#pragma unroll
                    for (int i = 0; i < XV / 16; ++i) store16(xp + 16 * i, x + 4 * i);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    top_z = word_max<T>(top_z, z[i]);
                    if (KIND == kClippedRef) top_x = word_max<T>(top_x, x[i]);
                }
            }
        }
        Sums q;
        q.m = warp_max_nan(word_top<T>(top_z));
        q.c = KIND == kClippedRef ? warp_max_nan(word_top<T>(top_x)) : -kInf;
        q.s = q.t = q.a = q.b = 0.f;
        q.za = -kInf;
        if (WARP) {
            __syncwarp();
        } else {
            if (lane == 0) { top_of[turn][warp][0] = q.m; top_of[turn][warp][1] = q.c; }
            __syncthreads();
            if (ALIKE && last_slot >= 0) {
                // every thread is done with the row before: its slot takes the next one
                const long long next = row + (sh.slots - 1) * step;
                if (next < r.n) {
                    fill(next, last_slot, ahead);
                    if (tid == 0) ahead = scalars_of(next + step);
                }
            }
            const int i = lane < warps ? lane : 0;
            q.m = warp_max_nan(top_of[turn][i][0]);
            if (KIND == kClippedRef) q.c = warp_max_nan(top_of[turn][i][1]);
        }
        if (live && act_e >= 0 && act_e / V >= v0 && act_e / V < p.v1 && (!r.bits || (ms[(act >> 5) - mask_first] >> (act & 31)) & 1u)) {
            const float v = to_f32(((const T*)zs)[act_e - v0 * V]);
            q.za = v == -kInf ? -3.4e38f : v;
        }

        // the sums
        if (live && q.m != -kInf) {
            const f32x2 M = pair(-q.m, -q.m), C = q.c == -kInf ? pair(0.f, 0.f) : pair(-q.c, -q.c), L = pair(kLog2e, kLog2e), minus = pair(-1.f, -1.f);
            f32x2 s = 0, t = 0, a = 0, b = 0;
#pragma unroll 2
            for (int v = v0 + tid; v < p.v1; v += team) {
                uint32_t z[4], x[XV / 4];
                load16(zs + (v - v0) * 16, z);
                if (KIND != kClipped)
#pragma unroll
                    for (int i = 0; i < XV / 16; ++i) load16(xs + (v - v0) * XV + 16 * i, x + 4 * i);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const f32x2 d = add2(elements<T>(z, i), M), e = ex2_2(mul2(d, L)), dl = floor2(d);
                    s = add2(s, e);
                    t = fma2(e, dl, t);
                    if (KIND == kSearch) {
                        const f32x2 y = elements<float>(x, i);
                        a = fma2(y, dl, a);
                        b = add2(b, y);
                    }
                    if (KIND == kClippedRef) {
                        const f32x2 c = add2(elements<T>(x, i), C);
                        b = add2(b, ex2_2(mul2(c, L)));
                        a = fma2(e, fma2(floor2(c), minus, dl), a);
                    }
                }
            }
            q.s = sum2(s); q.t = sum2(t); q.a = sum2(a); q.b = sum2(b);
        }
        if (live) {                              // the same in the whole team
            q.s = warp_sum(q.s);
            q.t = warp_sum(q.t);
            if (KIND != kClipped) { q.a = warp_sum(q.a); q.b = warp_sum(q.b); }
        }
        if (!WARP && live) {
            // every warp of the team leaves its sums with every CTA, and each warp joins them all, a lane an entry
            float (*to)[8] = part[part_turn];
            part_turn ^= 1;                      // only where a barrier follows: the other CTAs may still read the last ones
            if (lane < (int)ctas) {
                const uint32_t here = ptx::smem_u32(to[cta * warps + warp]);
                uint32_t there;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(lane));
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there), "f"(q.m), "f"(q.c), "f"(q.s), "f"(q.t) : "memory");
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there + 16), "f"(q.a), "f"(q.b), "f"(q.za), "f"(0.f) : "memory");
            }
            if (ctas == 1) __syncthreads();
            else cluster_barrier();
            const int parts = (int)ctas * warps;
            float M = -kInf, C = -kInf;
            if (ctas == 1) {
                M = q.m; C = q.c;
            } else {
                for (int i = lane; i < parts; i += 32) { M = max_nan(M, to[i][0]); C = max_nan(C, to[i][1]); }
                M = warp_max_nan(M);
                C = warp_max_nan(C);
            }
            q.s = q.t = q.a = q.b = 0.f;
            for (int i = lane; i < parts; i += 32) {
                float4 lo = *(const float4*)to[i];
                const float4 hi = *(const float4*)(to[i] + 4);
                if (ctas > 1) {
                    // a CTA's sums are relative to its own maxima
                    const float d = lo.x == -kInf ? 0.f : lo.x - M, c = lo.y == -kInf ? 0.f : lo.y - C;
                    const float f = lo.x == -kInf ? 0.f : ex2(d * kLog2e);
                    lo.z *= f;
                    lo.w = fmaf(d, lo.z, lo.w * f);
                    if (KIND == kSearch) q.a += fmaf(d, hi.y, hi.x);
                    if (KIND == kClippedRef) { q.a += fmaf(d - c, lo.z, hi.x * f); q.b = fmaf(hi.y, lo.y == -kInf ? 0.f : ex2(c * kLog2e), q.b); }
                } else {
                    q.a += hi.x;
                    if (KIND == kClippedRef) q.b += hi.y;
                }
                if (KIND == kSearch) q.b += hi.y;
                q.s += lo.z;
                q.t += lo.w;
                q.za = max_nan(q.za, hi.z);
            }
            q.s = warp_sum(q.s);
            q.t = warp_sum(q.t);
            if (KIND != kClipped) { q.a = warp_sum(q.a); q.b = warp_sum(q.b); }
            if (KIND != kSearch) q.za = warp_max_nan(q.za);
            q.m = M; q.c = C;
        }
        turn ^= 1;
        live = live && row_result<KIND>(r, q, w, scalars.y, scalars.z, &g, &out);
        if (tid == 0 && cta == 0) {
            if (r.loss) r.loss[row] = out.loss;
            if (r.stats) r.stats[row] = out.stats;
        }

        // the gradient
        T* grad = (T*)r.grad + row * r.g_pitch - p.head;
        const f32x2 M = pair(-g.M, -g.M), C = pair(-g.C, -g.C), L = pair(kLog2e, kLog2e), minus = pair(-1.f, -1.f);
        const f32x2 lp = pair(g.lp, g.lp), k0 = pair(g.k0, g.k0), kz = pair(g.kz, g.kz), kd = pair(g.kd, g.kd), kt = pair(-g.kt, -g.kt);
#pragma unroll 2
        for (int v = v0 + tid; v < p.v1; v += team) {
            uint32_t z[4] = {0, 0, 0, 0}, x[XV / 4];
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = 0.f;
            if (live) {
                load16(zs + (v - v0) * 16, z);
                if (KIND != kClipped)
#pragma unroll
                    for (int i = 0; i < XV / 16; ++i) load16(xs + (v - v0) * XV + 16 * i, x + 4 * i);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const f32x2 d = add2(elements<T>(z, i), M), pr = ex2_2(fma2(d, L, lp)), dl = floor2(d);
                    f32x2 y = fma2(kz, dl, k0);
                    if (KIND == kClippedRef) y = fma2(kd, fma2(floor2(add2(elements<T>(x, i), C)), minus, dl), y);
                    y = mul2(y, pr);
                    if (KIND == kSearch) y = fma2(kt, elements<float>(x, i), y);
                    halves(y, o[2 * i], o[2 * i + 1]);
                }
                if (KIND != kSearch && (unsigned)act_e - (unsigned)(v * V) < (unsigned)V)
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (act_e == v * V + i) o[i] += g.ka;
            }
            if (sizeof(T) == 4)
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = __float_as_uint(o[i % V]);
            else
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = pack2<T>(o[(2 * i) % V], o[(2 * i + 1) % V]);
            if (ALIKE) {
                const int e = v * V;
                if (e >= p.head && e + V <= p.head + r.A) {
                    *(uint4*)(grad + e) = make_uint4(z[0], z[1], z[2], z[3]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (e + i >= p.head && e + i < p.head + r.A) grad[e + i] = from_f32<T>(o[i]);
                }
            } else {
                store16(zs + (v - v0) * 16, z);
            }
        }
        // the slot's next copy comes behind what was read and written here
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (!ALIKE) {
            if (WARP) __syncwarp(); else __syncthreads();
            const int j1 = min(p.v1 * V, r.A);
            for (int j = v0 * V + tid; j < j1; j += team) grad[j] = ((const T*)zs)[j - v0 * V];
            if (WARP) __syncwarp(); else __syncthreads();
        } else if (WARP) {
            __syncwarp();
            const long long next = row + sh.slots * step;
            if (next < r.n) {
                fill(next, slot, ahead);
                if (tid == 0) ahead = scalars_of(next + step);
            }
        }
        last_slot = slot;
        if (++slot == sh.slots) { slot = 0; parity ^= 1; }
    }
    if (ALIKE && abort_flag) {                   // a wait ran out: what is still in flight is waited for once more, within the same limit
        int none = 0;
        for (int s = 0; s < sh.slots; ++s) ptx::mbar_wait(bars + 8 * s, s >= slot ? parity : parity ^ 1, &none);
    }
    // and none may leave while another may still write
    if (!WARP && ctas > 1) cluster_barrier();
}

// ---- rows of any length -----------------------------------------------------------
// Rows too long for the shared memory of eight CTAs (from some 200,000 actions on): a CTA goes over its row in device
// memory three times.
template <typename T, int KIND>
__global__ void __launch_bounds__(512)
policy_long_rows_kernel(const __grid_constant__ PolicyRows r) {
    const long long row = blockIdx.x;
    const T* z = (const T*)r.z + row * r.z_pitch;
    const uint8_t* x = (const uint8_t*)r.x + row * r.x_pitch * (KIND == kSearch ? 4 : sizeof(T));
    T* grad = (T*)r.grad + row * r.g_pitch;
    const uint32_t* bits = r.bits ? r.bits + row * r.mask_words : nullptr;
    const float w = r.weight ? r.weight[row] : 1.f;
    const int act = KIND == kSearch ? -1 : r.action[row], lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    auto second = [&](int j) { return KIND == kSearch ? target_f32(((const uint32_t*)x)[j], r.visits) : KIND == kClippedRef ? to_f32(((const T*)x)[j]) : 0.f; };
    __shared__ float part[2][16][8];
    bool live = w != 0.f;
    Sums q{-kInf, -kInf, 0.f, 0.f, 0.f, 0.f, -kInf};
    if (live)
        for (int j = threadIdx.x; j < r.A; j += 512)
            if (legal(bits, j)) {
                const float v = to_f32(z[j]);
                q.m = max_nan(q.m, v);
                if (KIND == kClippedRef) q.c = max_nan(q.c, second(j));
                if (KIND != kSearch && j == act) q.za = v == -kInf ? -3.4e38f : v;
            }
    q.m = warp_max_nan(q.m); q.c = warp_max_nan(q.c); q.za = warp_max_nan(q.za);
    if (lane == 0) { part[0][warp][0] = q.m; part[0][warp][1] = q.c; part[0][warp][2] = q.za; }
    __syncthreads();
    q.m = warp_max_nan(part[0][lane % 16][0]); q.c = warp_max_nan(part[0][lane % 16][1]); q.za = warp_max_nan(part[0][lane % 16][2]);
    const float C = q.c == -kInf ? 0.f : q.c;
    live = live && q.m != -kInf;                 // the same in the whole CTA
    if (live)
        for (int j = threadIdx.x; j < r.A; j += 512)
            if (legal(bits, j)) {
                const float d = to_f32(z[j]) - q.m, e = ex2(d * kLog2e), dl = fmaxf(d, kLow), y = second(j);
                q.s += e;
                q.t = fmaf(e, dl, q.t);
                if (KIND == kSearch) { q.a = fmaf(y, dl, q.a); q.b += y; }
                if (KIND == kClippedRef) { q.a = fmaf(e, dl - fmaxf(y - C, kLow), q.a); q.b += ex2((y - C) * kLog2e); }
            }
    q.s = warp_sum(q.s); q.t = warp_sum(q.t); q.a = warp_sum(q.a); q.b = warp_sum(q.b);
    if (lane == 0) { part[1][warp][0] = q.s; part[1][warp][1] = q.t; part[1][warp][2] = q.a; part[1][warp][3] = q.b; }
    __syncthreads();
    const float* from = part[1][lane % 16];      // each entry by two lanes
    q.s = 0.5f * warp_sum(from[0]); q.t = 0.5f * warp_sum(from[1]); q.a = 0.5f * warp_sum(from[2]); q.b = 0.5f * warp_sum(from[3]);
    RowGrad g;
    RowOut out{0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    live = live && row_result<KIND>(r, q, w, KIND == kSearch ? 0.f : r.old_logp[row], KIND == kSearch ? 0.f : r.advantage[row], &g, &out);
    if (threadIdx.x == 0) {
        if (r.loss) r.loss[row] = out.loss;
        if (r.stats) r.stats[row] = out.stats;
    }
    for (int j = threadIdx.x; j < r.A; j += 512) {
        float o = 0.f;
        if (live && legal(bits, j)) {
            const float d = to_f32(z[j]) - g.M, dl = fmaxf(d, kLow), y = second(j);
            o = fmaf(g.kz, dl, g.k0);
            if (KIND == kClippedRef) o = fmaf(g.kd, dl - fmaxf(y - g.C, kLow), o);
            o *= ex2(fmaf(d, kLog2e, g.lp));
            if (KIND == kSearch) o = fmaf(-g.kt, y, o);
            else if (j == act) o += g.ka;
        }
        grad[j] = from_f32<T>(o);
    }
}

// ---- host ---------------------------------------------------------------------------
constexpr int kMostShared = 200 * 1024;          // of a CTA; 227 KB less the kernel's own

template <typename T, int KIND, bool WARP, bool ALIKE>
int launch_kernel(const PolicyRows& r, RowShape sh, int threads, int ctas, cudaStream_t st) {
    auto kernel = policy_rows_kernel<T, KIND, WARP, ALIKE>;
    static std::atomic<int> known{0};            // registers of a thread | SMs << 16, once looked up; every device is of the same kind
    int k = known.load(std::memory_order_acquire);
    if (!k) {
        int dev = 0, sms = 0;
        cudaFuncAttributes a;
        OB200_CUDA_OK(cudaGetDevice(&dev));
        OB200_CUDA_OK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        OB200_CUDA_OK(cudaFuncGetAttributes(&a, kernel));
        OB200_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
        k = a.numRegs | sms << 16;
        known.store(k, std::memory_order_release);
    }
    const int smem = WARP ? sh.team_bytes * threads / 32 : sh.team_bytes;
    const int by_regs = 65536 / (((k & 0xFFFF) + 7) / 8 * 8 * threads), by_smem = 224 * 1024 / (smem + 10 * 1024), by_threads = 2048 / threads;
    int per_sm = by_regs < by_smem ? by_regs : by_smem;
    per_sm = per_sm < by_threads ? per_sm : by_threads;
    if (per_sm < 1) per_sm = 1;
    const long long room = (long long)(k >> 16) * per_sm / ctas, teams = WARP ? (r.n + threads / 32 - 1) / (threads / 32) : r.n;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)ctas, 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((teams < room ? teams : room) * ctas));
    cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = ctas > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, r, sh);
    OB200_LAUNCHED("policy_rows_kernel");
    return OB200_OK;
}

template <typename T, int KIND, bool ALIKE>
int launch_shape(const PolicyRows& r, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T), XV = KIND == kClipped ? 0 : V * (KIND == kSearch ? 4 : (int)sizeof(T));
    const int vecs = (int)(((long long)r.A + (ALIKE ? V - 1 : 0) + V - 1) / V);
    RowShape sh{};
    sh.error = device_error_word();
    if (!sh.error) return set_error(OB200_ERR_CUDA, "policy loss: the device's error word is not available");
    auto lay = [&](int ctas) {                   // fills sh but for the slots; the bytes of a slot
        sh.seg = (vecs + ctas - 1) / ctas;
        sh.x_at = 16 + sh.seg * 16;
        sh.mask_at = sh.x_at + sh.seg * XV;
        sh.slot_bytes = (sh.mask_at + (r.bits ? (sh.seg * V / 32 + 2) * 4 : 0) + 15) / 16 * 16;
        return sh.slot_bytes;
    };
    auto finish = [&](int slots) {
        sh.slots = slots;
        sh.team_bytes = (slots * (sh.slot_bytes + 8) + 127) / 128 * 128;
        return sh.team_bytes;
    };
    if (r.A <= 1024) {
        lay(1);
        const int fit = 72 * 1024 / finish(2), warps = fit < 1 ? 1 : fit > 8 ? 8 : fit;
        return launch_kernel<T, KIND, true, ALIKE>(r, sh, 32 * warps, 1, st);
    }
    if ((long long)vecs * (16 + XV) <= 8LL * kMostShared / 2) {
        int ctas = 1;
        while (ctas < 8 && lay(ctas) > 36 * 1024) ctas *= 2;
        if (2 * (lay(ctas) + 8) + 128 <= kMostShared) {
            finish(sh.slot_bytes <= 20 * 1024 ? 3 : 2);
            int threads = (sh.seg / 8 + 31) / 32 * 32;
            threads = threads < 64 ? 64 : threads > 512 ? 512 : threads;
            return launch_kernel<T, KIND, false, ALIKE>(r, sh, threads, ctas, st);
        }
    }
    policy_long_rows_kernel<T, KIND><<<(unsigned)r.n, 512, 0, st>>>(r);
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

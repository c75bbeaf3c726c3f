// Policy losses over rows of logits, with their gradients: cross entropy with the search's visit distribution, and the
// clipped-ratio loss with a KL term against a reference policy.
//
// With M the largest legal logit, e_j = exp(z_j - M), s = sum e, t = sum e (z - M), p_j = e_j / s, both gradients need no
// more than sums over the row:
//   H(p) = log s - t / s                                 dH/dz_j  = -p_j ((z_j - M) - t / s)
//   KL(p|q) = u / s - (lse(z) - lse(q's logits)),  u = sum e (z - zq)
//                                                        dKL/dz_j = p_j ((z_j - zq_j) - u / s)
//   cross entropy = log s - c / T,  c = sum target (z - M), T = sum target
//                                                        d/dz_j   = p_j - target_j / T
//   clipped term: d/dz_j = k ([j = action] - p_j),  k = -advantage r or 0
// so a gradient is p_j (k0 + kz (z_j - M) + kd (z_j - zq_j)) plus a term of the action or of the target.
#include "common.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace ob200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

enum Kind { kVisits = 0, kProbs = 1, kClipped = 2, kClippedRef = 3 };

struct Rows {
    const void* z; const void* x;       // logits; target or reference logits
    const uint32_t* bits; const float* weight;
    void* grad; float* loss; float4* stats;
    long long z_pitch, x_pitch, g_pitch;
    int n, A, mask_words;
    // search: entropy; clipped: all of it
    const int32_t* action; const float* old_logp; const float* advantage;
    float entropy, kl, lo, hi;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(int32_t v) { return (float)v; }
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
// exp(z - m), the difference first: rows whose logits all stand at the type's lowest value are uniform, not NaN
__device__ __forceinline__ float exp_from(float z, float m) { return ex2((z - m) * kLog2e); }

// Sums of a part of a row, relative to the part's largest legal logit m (-inf: no legal action).
// a, b: search: sum target (z - m), sum target;  clipped: u, and the reference row's sum of exp relative to its maximum c.
template <int KIND>
struct Sums {
    float m = -kInf, s = 0.f, t = 0.f, a = 0.f, b = 0.f, c = -kInf;

    __device__ __forceinline__ void rebase(float M) {
        // a part without a legal action has nothing to scale, and its m no difference
        const float d = m == -kInf ? 0.f : m - M, f = m == -kInf ? 0.f : ex2(d * kLog2e);
        s *= f;
        t = fmaf(d, s, t * f);               // d may be as low as -3.4e38: it meets s after f has
        if (KIND == kVisits || KIND == kProbs) a += d * b;
        else a *= f;
        m = M;
    }
    __device__ __forceinline__ void rebase_ref(float C) {
        b *= c == -kInf ? 0.f : ex2((c - C) * kLog2e);
        c = C;
    }
    __device__ __forceinline__ void add(float z, float x) {
        if (z > m) rebase(z);
        const float e = exp_from(z, m), d = z - m;
        s += e;
        t = fmaf(e, d, t);
        if (KIND == kVisits || KIND == kProbs) { a = fmaf(x, d, a); b += x; }
        if (KIND == kClippedRef) {
            if (x > c) rebase_ref(x);
            a = fmaf(e, e == 0.f ? 0.f : z - x, a);
            b += x == -kInf ? 0.f : exp_from(x, c);
        }
    }
    __device__ __forceinline__ void join(Sums o) {
        const float M = fmaxf(m, o.m);
        rebase(M); o.rebase(M);
        s += o.s; t += o.t; a += o.a;
        if (KIND == kClippedRef) {
            const float C = fmaxf(c, o.c);
            rebase_ref(C); o.rebase_ref(C);
        }
        b += o.b;
    }
    __device__ __forceinline__ Sums shuffled(int lane_mask) const {
        Sums o;
        o.m = __shfl_xor_sync(~0u, m, lane_mask); o.s = __shfl_xor_sync(~0u, s, lane_mask);
        o.t = __shfl_xor_sync(~0u, t, lane_mask); o.a = __shfl_xor_sync(~0u, a, lane_mask);
        o.b = __shfl_xor_sync(~0u, b, lane_mask);
        o.c = KIND == kClippedRef ? __shfl_xor_sync(~0u, c, lane_mask) : -kInf;
        return o;
    }
};

// What the second look at a row needs: gradient = p (k0 + kz (z - M) + kd (z - x)) + ka [action] - kt target.
struct RowGrad { float M, inv_s, k0, kz, kd, ka, kt; };
struct RowOut { float loss; float4 stats; };

// live: the row has not been left out for its weight or action.  False when the row is left out.
template <int KIND>
__device__ __forceinline__ bool row_result(const Rows& r, const Sums<KIND>& q, int row, float w, float z_action, RowGrad* g, RowOut* o) {
    if (q.s == 0.f) return false;
    const float ls = logf(q.s), inv_s = 1.f / q.s, mean = q.t * inv_s, H = ls - mean;
    g->M = q.m; g->inv_s = inv_s;
    g->kz = w * r.entropy; g->kd = 0.f; g->ka = 0.f; g->kt = 0.f;
    if (KIND == kVisits || KIND == kProbs) {
        if (!(q.b != 0.f)) return false;
        const float inv_T = 1.f / q.b, ce = ls - q.a * inv_T;
        g->k0 = w * (1.f - r.entropy * mean);
        g->kt = w * inv_T;
        o->loss = w * (ce - r.entropy * H);
        o->stats = make_float4(ce, H, q.b, q.m + ls);
        return true;
    }
    const float logp = (z_action - q.m) - ls, adv = r.advantage[row];
    const float ratio = expf(logp - r.old_logp[row]);
    float surrogate = 0.f, k = 0.f;
    if (adv != 0.f) {
        const float open = ratio * adv, held = fminf(fmaxf(ratio, r.lo), r.hi) * adv;
        surrogate = open <= held ? open : held;
        k = open <= held ? -open : 0.f;
        if (ratio != ratio || adv != adv) surrogate = k = open;
    }
    float kl = 0.f, ud = 0.f;
    if (KIND == kClippedRef) {
        ud = q.a * inv_s;
        kl = ud - ((q.m - q.c) + (ls - logf(q.b)));
    }
    g->k0 = w * (-k - r.kl * ud - r.entropy * mean);
    g->kd = w * r.kl;
    g->ka = w * k;
    o->loss = w * (-surrogate + r.kl * kl - r.entropy * H);
    o->stats = make_float4(logp, ratio, kl, H);
    return true;
}

__device__ __forceinline__ bool legal(const uint32_t* bits, int j) { return !bits || (bits[j >> 5] >> (j & 31)) & 1u; }

// TEAM threads (a warp, or the whole CTA of 256) go over a row twice: once for the sums, once for the gradient.
template <typename T, int KIND, int TEAM>
__global__ void __launch_bounds__(256)
policy_loss_kernel(const Rows r) {
    using X = typename std::conditional<KIND == kVisits, int32_t, typename std::conditional<KIND == kProbs, float, T>::type>::type;
    constexpr bool kClip = KIND == kClipped || KIND == kClippedRef, kSecond = KIND != kClipped;
    const int rank = threadIdx.x % TEAM;
    const long long row = (long long)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM;
    if (row >= r.n) return;
    const T* z = (const T*)r.z + row * r.z_pitch;
    const X* x = (const X*)r.x + row * r.x_pitch;
    T* grad = (T*)r.grad + row * r.g_pitch;
    const uint32_t* bits = r.bits ? r.bits + row * r.mask_words : nullptr;
    const float w = r.weight ? r.weight[row] : 1.f;
    bool live = w != 0.f;
    int act = -1;
    float z_act = 0.f;
    if (kClip && live) {
        act = r.action[row];
        live = act >= 0 && act < r.A && legal(bits, act);
        if (live) { z_act = to_f32(z[act]); live = z_act != -kInf; }
    }
    Sums<KIND> q;
    if (live)
        for (int j = rank; j < r.A; j += TEAM) {
            const float zj = to_f32(z[j]);
            if (zj != -kInf && legal(bits, j)) q.add(zj, kSecond ? to_f32(x[j]) : 0.f);
        }
#pragma unroll
    for (int o = 16; o; o >>= 1) q.join(q.shuffled(o));
    if (TEAM > 32) {
        __shared__ float part[8][6];
        if (threadIdx.x % 32 == 0) {
            float* to = part[threadIdx.x / 32];
            to[0] = q.m; to[1] = q.s; to[2] = q.t; to[3] = q.a; to[4] = q.b; to[5] = q.c;
        }
        __syncthreads();
        const float* from = part[threadIdx.x % 8];
        q.m = from[0]; q.s = from[1]; q.t = from[2]; q.a = from[3]; q.b = from[4]; q.c = from[5];
#pragma unroll
        for (int o = 4; o; o >>= 1) q.join(q.shuffled(o));
    }
    RowGrad g;
    RowOut out{0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    live = live && row_result<KIND>(r, q, (int)row, w, z_act, &g, &out);
    if (rank == 0) {
        if (r.loss) r.loss[row] = out.loss;
        if (r.stats) r.stats[row] = out.stats;
    }
    for (int j = rank; j < r.A; j += TEAM) {
        float v = 0.f;
        if (live) {
            const float zj = to_f32(z[j]);
            if (zj != -kInf && legal(bits, j)) {
                const float xj = kSecond ? to_f32(x[j]) : 0.f;
                const float p = exp_from(zj, g.M) * g.inv_s;
                if (p != 0.f) {
                    v = fmaf(g.kz, zj - g.M, g.k0);
                    if (KIND == kClippedRef && g.kd != 0.f) v = fmaf(g.kd, zj - xj, v);
                    v *= p;
                }
                if (kClip) { if (j == act) v += g.ka; }
                else v = fmaf(-g.kt, xj, v);
            }
        }
        grad[j] = from_f32<T>(v);
    }
}

template <typename T, int KIND>
int launch_typed(const Rows& r, cudaStream_t st) {
    if (r.A <= 1024) policy_loss_kernel<T, KIND, 32><<<(unsigned)((r.n + 7) / 8), 256, 0, st>>>(r);
    else policy_loss_kernel<T, KIND, 256><<<(unsigned)r.n, 256, 0, st>>>(r);
    OB200_LAUNCHED("policy_loss_kernel");
    return OB200_OK;
}

template <int KIND>
int launch_kind(const Rows& r, int dtype, cudaStream_t st) {
    if (dtype == OB200_DTYPE_BF16) return launch_typed<__nv_bfloat16, KIND>(r, st);
    if (dtype == OB200_DTYPE_F16) return launch_typed<__half, KIND>(r, st);
    return launch_typed<float, KIND>(r, st);
}

int elem_bytes(int dtype) { return dtype == OB200_DTYPE_F32 ? 4 : 2; }

// Whether rows [n][A] of `es`-byte elements at a (pitch pa) and of eb-byte elements at b (pitch pb) may share a byte.
bool rows_meet(const void* a, long long pa, int ea, const void* b, long long pb, int eb, long long n, long long A) {
    const intptr_t a0 = (intptr_t)a, b0 = (intptr_t)b;
    const intptr_t a1 = a0 + ((n - 1) * pa + A) * ea, b1 = b0 + ((n - 1) * pb + A) * eb;
    if (a1 <= b0 || b1 <= a0) return false;
    if (pa * ea != pb * eb) return true;
    const intptr_t step = pa * ea, off = (((b0 - a0) % step) + step) % step;   // b's rows start here within a's
    return off < A * ea || off + A * eb > step;
}

// What both losses ask of their rows; fills the shared part of r.
int take_rows(const char* who, const ob200_policy_rows* p, Rows* r) {
    if (!p) return set_error(OB200_ERR_INVALID, "%s: null argument", who);
    if (p->dtype != OB200_DTYPE_BF16 && p->dtype != OB200_DTYPE_F16 && p->dtype != OB200_DTYPE_F32)
        return set_error(OB200_ERR_INVALID, "%s: bad dtype %d", who, p->dtype);
    if (p->n < 0 || p->n_actions < 1) return set_error(OB200_ERR_INVALID, "%s: bad size (n %d, n_actions %d)", who, p->n, p->n_actions);
    if (p->n == 0) return OB200_OK;
    const int es = elem_bytes(p->dtype);
    if (!p->logits || !p->grad) return set_error(OB200_ERR_INVALID, "%s: null logits or grad", who);
    if (p->logits_pitch < p->n_actions || p->grad_pitch < p->n_actions)
        return set_error(OB200_ERR_INVALID, "%s: a pitch is below n_actions", who);
    if (((uintptr_t)p->logits | (uintptr_t)p->grad) % es || ((uintptr_t)p->legal_bits | (uintptr_t)p->row_weight | (uintptr_t)p->loss) % 4 || (uintptr_t)p->stats % 16)
        return set_error(OB200_ERR_INVALID, "%s: a pointer is not aligned", who);
    if (p->legal_bits && p->mask_words < (p->n_actions + 31) / 32)
        return set_error(OB200_ERR_INVALID, "%s: mask_words %d too small for %d actions", who, p->mask_words, p->n_actions);
    if (!(p->grad == p->logits && p->grad_pitch == p->logits_pitch) &&
        rows_meet(p->grad, p->grad_pitch, es, p->logits, p->logits_pitch, es, p->n, p->n_actions))
        return set_error(OB200_ERR_INVALID, "%s: grad overlaps logits (it may be logits itself, with the same pitch)", who);
    r->z = p->logits; r->bits = p->legal_bits; r->weight = p->row_weight;
    r->grad = p->grad; r->loss = p->loss; r->stats = (float4*)p->stats;
    r->z_pitch = p->logits_pitch; r->g_pitch = p->grad_pitch;
    r->n = p->n; r->A = p->n_actions; r->mask_words = p->mask_words;
    return OB200_OK;
}

}  // namespace
}  // namespace ob200

using namespace ob200;

extern "C" {

int ob200_launch_policy_loss_search(const ob200_policy_rows* rows, const void* target, int64_t target_pitch, int32_t target_kind,
                                    float entropy_coef, ob200_stream stream) {
    const char* who = "ob200_launch_policy_loss_search";
    Rows r{};
    if (int rc = take_rows(who, rows, &r)) return rc;
    if (target_kind != OB200_TARGET_VISITS && target_kind != OB200_TARGET_PROBS)
        return set_error(OB200_ERR_INVALID, "%s: bad target_kind %d", who, target_kind);
    if (rows->n > 0) {
        if (!target || (uintptr_t)target % 4 || target_pitch < r.A)
            return set_error(OB200_ERR_INVALID, "%s: target is null, not aligned, or its pitch is below n_actions", who);
        if (rows_meet(r.grad, r.g_pitch, elem_bytes(rows->dtype), target, target_pitch, 4, r.n, r.A))
            return set_error(OB200_ERR_INVALID, "%s: grad overlaps target", who);
    }
    if (int rc = require_device()) return rc;
    if (rows->n == 0) return OB200_OK;
    r.x = target; r.x_pitch = target_pitch; r.entropy = entropy_coef;
    return target_kind == OB200_TARGET_VISITS ? launch_kind<kVisits>(r, rows->dtype, as_stream(stream))
                                              : launch_kind<kProbs>(r, rows->dtype, as_stream(stream));
}

int ob200_launch_policy_loss_clipped(const ob200_policy_rows* rows, const int32_t* action, const float* old_logp, const float* advantage,
                                     const void* ref_logits, int64_t ref_pitch, float clip_low, float clip_high, float kl_coef,
                                     float entropy_coef, ob200_stream stream) {
    const char* who = "ob200_launch_policy_loss_clipped";
    Rows r{};
    if (int rc = take_rows(who, rows, &r)) return rc;
    if (!(clip_low >= 0.f) || !(clip_high >= 0.f)) return set_error(OB200_ERR_INVALID, "%s: a clip range is negative", who);
    if (!ref_logits && kl_coef != 0.f) return set_error(OB200_ERR_INVALID, "%s: kl_coef without ref_logits", who);
    if (rows->n > 0) {
        if (!action || !old_logp || !advantage || ((uintptr_t)action | (uintptr_t)old_logp | (uintptr_t)advantage) % 4)
            return set_error(OB200_ERR_INVALID, "%s: action, old_logp or advantage is null or not aligned", who);
        if (ref_logits) {
            const int es = elem_bytes(rows->dtype);
            if ((uintptr_t)ref_logits % es || ref_pitch < r.A)
                return set_error(OB200_ERR_INVALID, "%s: ref_logits is not aligned or its pitch is below n_actions", who);
            if (rows_meet(r.grad, r.g_pitch, es, ref_logits, ref_pitch, es, r.n, r.A))
                return set_error(OB200_ERR_INVALID, "%s: grad overlaps ref_logits", who);
        }
    }
    if (int rc = require_device()) return rc;
    if (rows->n == 0) return OB200_OK;
    r.x = ref_logits; r.x_pitch = ref_pitch;
    r.action = action; r.old_logp = old_logp; r.advantage = advantage;
    r.lo = 1.f - clip_low; r.hi = 1.f + clip_high; r.kl = kl_coef; r.entropy = entropy_coef;
    return ref_logits ? launch_kind<kClippedRef>(r, rows->dtype, as_stream(stream)) : launch_kind<kClipped>(r, rows->dtype, as_stream(stream));
}

}  // extern "C"

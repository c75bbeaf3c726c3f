// The weight update: the 2-norm of all gradients of a network with the factor that clips it, and one AdamW step over all
// its tensors, states in fp32 or in e4m3 with a scale per 256 elements.
//
// Both go over the tensors in chunks of 2,048 elements, a CTA each; the list of tensors travels as a kernel parameter
// (up to 32 KB), so that a call needs no device table, no copy and no memory of its own and can be captured.
#include "common.h"
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace ob200 {
namespace {

constexpr int kBlock = 256;              // elements that share the scales of 8-bit states
constexpr int kChunk = 2048;             // elements of a CTA: eight warps, a block each
constexpr float kE4m3Max = 448.f, kE4m3Least = 0x1p-9f, kScaleFloor = 0x1p-110f;
constexpr int kNormCtas = 592;           // partial sums of the norm: four CTAs per SM

struct Entry {
    void* p; const void* g; void* m; void* v;
    float *ms, *vs;
    long long n;
    int chunk0;                          // first chunk of this tensor within the launch
    float decay;
};
template <int N> struct Table { int count, chunks; Entry e[N]; };
constexpr int kSmallTable = 48, kLargeTable = 500;
static_assert(sizeof(Table<kLargeTable>) + 128 <= 32764, "the table has to fit the kernel parameters");

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// The tensor that holds a chunk: the last one whose first chunk is not behind it (tensors without elements are not listed).
template <int N>
__device__ __forceinline__ const Entry& entry_of(const Table<N>& t, int chunk) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].chunk0 <= chunk) lo = mid; else hi = mid - 1;
    }
    return t.e[lo];
}

// ---- norm ----------------------------------------------------------------------
// Squares and a thread's sums in fp32 (a thread sees a few hundred elements), everything beyond a thread in fp64.
template <typename G, int N>
__global__ void __launch_bounds__(256)
grad_norm_part_kernel(const __grid_constant__ Table<N> t, double* __restrict__ part) {
    double sum = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Entry& e = entry_of(t, c);
        const long long at = (long long)(c - e.chunk0) * kChunk;
        const G* g = (const G*)e.g;
        float s = 0.f;
        for (int i = threadIdx.x; i < kChunk && at + i < e.n; i += 256) {
            const float v = to_f32(g[at + i]);
            s = fmaf(v, v, s);
        }
        sum += (double)s;
    }
    __shared__ double warp_sum[8];
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double a = 0.0;
        for (int w = 0; w < 8; ++w) a += warp_sum[w];
        part[blockIdx.x] = a;
    }
}

__global__ void __launch_bounds__(256)
grad_norm_finish_kernel(const double* __restrict__ part, int n, float max_norm, float* __restrict__ out) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) sum += part[i];
    __shared__ double warp_sum[8];
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x) return;
    double a = 0.0;
    for (int w = 0; w < 8; ++w) a += warp_sum[w];
    const double norm = sqrt(a);
    out[0] = (float)norm;
    // an infinite norm gives NaN, not 0: the step is to be left out, not made with zeroed gradients
    out[1] = !isfinite((float)norm) ? __int_as_float(0x7fc00000) : norm > (double)max_norm ? (float)((double)max_norm / norm) : 1.f;
}

// ---- AdamW ----------------------------------------------------------------------
struct Step {
    float lr, beta1, one_beta1, beta2, one_beta2, eps;
    float rate;                          // 1 / (1 - beta1^step)
    float root;                          // 1 / sqrt(1 - beta2^step)
    double beta1_d, beta2_d;
    const float* grad_scale; const float* lr_device; const int32_t* step_device;
};

__device__ __forceinline__ float decode_e4m3(uint8_t c) {
    __nv_fp8_e4m3 v;
    v.__x = c;
    return (float)v;
}
__device__ __forceinline__ uint8_t encode_e4m3(float x) { return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }

// Largest of the warp's non-negative values (NaN is larger than all).
__device__ __forceinline__ float warp_max(float v) { return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(v))); }

template <typename P, typename G, int BITS, int N>
__global__ void __launch_bounds__(256)
adamw_kernel(const __grid_constant__ Table<N> t, const __grid_constant__ Step k) {
    const float gs = k.grad_scale ? *k.grad_scale : 1.f;
    if (!isfinite(gs)) return;
    const float lr = k.lr_device ? *k.lr_device : k.lr;
    float rate = k.rate, root = k.root;
    if (k.step_device) {
        const double step = (double)*k.step_device;
        rate = (float)(1.0 / (1.0 - pow(k.beta1_d, step)));
        root = (float)(1.0 / sqrt(1.0 - pow(k.beta2_d, step)));
    }
    rate *= lr;
    const Entry& e = entry_of(t, blockIdx.x);
    const int lane = threadIdx.x % 32;
    const long long block = (long long)((int)blockIdx.x - e.chunk0) * (kChunk / kBlock) + threadIdx.x / 32;
    const long long at = block * kBlock;
    if (at >= e.n) return;
    const int left = (int)min((long long)kBlock, e.n - at);
    const float keep = fmaf(-lr, e.decay, 1.f);
    P* p = (P*)e.p + at;
    const G* g = (const G*)e.g + at;
    float ms = 0.f, vs = 0.f;
    if (BITS == 8) { ms = e.ms[block]; vs = e.vs[block]; }
    float mm[8], rr[8], m_top = 0.f, r_top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int j = lane + 32 * i;
        mm[i] = rr[i] = 0.f;
        if (j >= left) continue;
        float m, v;
        if (BITS == 32) { m = ((const float*)e.m)[at + j]; v = ((const float*)e.v)[at + j]; }
        else {
            m = __fmul_rn(decode_e4m3(((const uint8_t*)e.m)[at + j]), ms);
            const float r = __fmul_rn(decode_e4m3(((const uint8_t*)e.v)[at + j]), vs);
            v = __fmul_rn(r, r);
        }
        const float gr = __fmul_rn(to_f32(g[j]), gs);
        m = __fadd_rn(__fmul_rn(m, k.beta1), __fmul_rn(gr, k.one_beta1));
        v = __fadd_rn(__fmul_rn(v, k.beta2), __fmul_rn(__fmul_rn(gr, gr), k.one_beta2));
        const float r = __fsqrt_rn(v);
        p[j] = from_f32<P>(fmaf(-rate, __fdividef(m, fmaf(r, root, k.eps)), to_f32(p[j]) * keep));
        if (BITS == 32) { ((float*)e.m)[at + j] = m; ((float*)e.v)[at + j] = v; }
        mm[i] = m; rr[i] = r;
        m_top = __uint_as_float(max(__float_as_uint(m_top), __float_as_uint(fabsf(m))));
        r_top = __uint_as_float(max(__float_as_uint(r_top), __float_as_uint(fabsf(r))));
    }
    if (BITS == 8) {
        m_top = warp_max(m_top); r_top = warp_max(r_top);
        if (m_top < kScaleFloor) m_top = kScaleFloor;
        if (r_top < kScaleFloor) r_top = kScaleFloor;
        const float mi = __fdiv_rn(kE4m3Max, m_top), ri = __fdiv_rn(kE4m3Max, r_top);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int j = lane + 32 * i;
            if (j >= left) continue;
            ((uint8_t*)e.m)[at + j] = encode_e4m3(__fmul_rn(mm[i], mi));
            const float x = __fmul_rn(rr[i], ri);
            ((uint8_t*)e.v)[at + j] = encode_e4m3(rr[i] > 0.f && x < kE4m3Least ? kE4m3Least : x);
        }
        if (lane == 0) { e.ms[block] = __fdiv_rn(m_top, kE4m3Max); e.vs[block] = __fdiv_rn(r_top, kE4m3Max); }
    }
}

// ---- host ----------------------------------------------------------------------
int elem_bytes(int dtype) { return dtype == OB200_DTYPE_F32 ? 4 : 2; }
bool is_dtype(int d) { return d == OB200_DTYPE_BF16 || d == OB200_DTYPE_F16 || d == OB200_DTYPE_F32; }

// Fills t with tensors [*next, n) as far as they fit; false when there was nothing left to take.
template <int N>
bool fill_table(Table<N>* t, const ob200_train_tensor* in, int n, int* next, long long* chunks) {
    t->count = 0;
    *chunks = 0;
    for (; *next < n && t->count < N; ++*next) {
        const ob200_train_tensor& a = in[*next];
        if (a.numel == 0) continue;
        const long long c = (a.numel + kChunk - 1) / kChunk;
        if (t->count && *chunks + c > 0x7fffffffLL) break;   // the rest in another launch
        t->e[t->count++] = Entry{a.param, a.grad, a.exp_avg, a.exp_avg_sq, a.exp_avg_scale, a.exp_avg_sq_scale, a.numel, (int)*chunks, a.weight_decay};
        *chunks += c;
    }
    t->chunks = (int)*chunks;
    return t->count > 0;
}

constexpr long long kMostElements = 0x7fffffffLL * kChunk;

int check_list(const char* who, const ob200_train_tensor* t, int n) {
    if (n < 0 || (n > 0 && !t)) return set_error(OB200_ERR_INVALID, "%s: null tensors or a negative count", who);
    for (int i = 0; i < n; ++i) {
        if (t[i].numel < 0) return set_error(OB200_ERR_INVALID, "%s: tensor %d has a negative size", who, i);
        if (t[i].numel > kMostElements) return set_error(OB200_ERR_TOO_LARGE, "%s: tensor %d has over 2^42 elements", who, i);
        if (t[i].numel && !t[i].grad) return set_error(OB200_ERR_INVALID, "%s: tensor %d has no gradient", who, i);
    }
    return OB200_OK;
}

template <typename G, int N>
int norm_launches(const ob200_train_tensor* tensors, int n, double* part, int* parts, cudaStream_t st) {
    Table<N> t;
    int next = 0;
    long long chunks;
    while (fill_table(&t, tensors, n, &next, &chunks)) {
        // each launch its own partial sums; lists of more than one launch share the places out
        const int room = kNormCtas - *parts, more = (n - next + N - 1) / N;
        if (room < 1) return set_error(OB200_ERR_TOO_LARGE, "ob200_launch_grad_norm: too many tensors");
        const int ctas = (int)std::min<long long>(chunks, std::max(1, room / (1 + more)));
        grad_norm_part_kernel<G, N><<<ctas, 256, 0, st>>>(t, part + *parts);
        OB200_LAUNCHED("grad_norm_part_kernel");
        *parts += ctas;
    }
    return OB200_OK;
}

template <typename P, typename G, int BITS, int N>
int adamw_launches(const ob200_train_tensor* tensors, int n, const Step& k, cudaStream_t st) {
    Table<N> t;
    int next = 0;
    long long chunks;
    while (fill_table(&t, tensors, n, &next, &chunks)) {
        adamw_kernel<P, G, BITS, N><<<(unsigned)chunks, 256, 0, st>>>(t, k);
        OB200_LAUNCHED("adamw_kernel");
    }
    return OB200_OK;
}

template <typename P, typename G>
int adamw_typed(const ob200_train_tensor* tensors, int n, int bits, const Step& k, cudaStream_t st) {
    if (n <= kSmallTable)
        return bits == 8 ? adamw_launches<P, G, 8, kSmallTable>(tensors, n, k, st) : adamw_launches<P, G, 32, kSmallTable>(tensors, n, k, st);
    return bits == 8 ? adamw_launches<P, G, 8, kLargeTable>(tensors, n, k, st) : adamw_launches<P, G, 32, kLargeTable>(tensors, n, k, st);
}

template <typename P>
int adamw_param(const ob200_train_tensor* tensors, int n, const ob200_adamw_config* c, const Step& k, cudaStream_t st) {
    if (c->grad_dtype == OB200_DTYPE_BF16) return adamw_typed<P, __nv_bfloat16>(tensors, n, c->state_bits, k, st);
    if (c->grad_dtype == OB200_DTYPE_F16) return adamw_typed<P, __half>(tensors, n, c->state_bits, k, st);
    return adamw_typed<P, float>(tensors, n, c->state_bits, k, st);
}

// Whether two entries share memory of one kind (`base`, es bytes an element): two CTAs would update it at once.
int check_apart(const char* who, const ob200_train_tensor* t, int n, int es, void* ob200_train_tensor::*base, const char* what) {
    auto begin = [&](int i) { return (uintptr_t)(t[i].*base); };
    auto end = [&](int i) { return begin(i) + (uintptr_t)t[i].numel * es; };
    uintptr_t last = 0;
    bool apart = true;
    for (int i = 0; i < n && apart; ++i)
        if (t[i].numel) { apart = begin(i) >= last; last = end(i); }
    if (apart) return OB200_OK;           // in the order of memory, as the views of a flat buffer are
    std::unique_ptr<int[]> order(new (std::nothrow) int[n]);
    if (!order) return set_error(OB200_ERR_STATE, "%s: out of host memory", who);
    int k = 0;
    for (int i = 0; i < n; ++i)
        if (t[i].numel) order[k++] = i;
    std::sort(order.get(), order.get() + k, [&](int a, int b) { return begin(a) < begin(b); });
    for (int i = 1; i < k; ++i)
        if (begin(order[i]) < end(order[i - 1]))
            return set_error(OB200_ERR_INVALID, "%s: tensors %d and %d share memory (%s)", who, order[i - 1], order[i], what);
    return OB200_OK;
}

}  // namespace
}  // namespace ob200

using namespace ob200;

extern "C" {

int64_t ob200_grad_norm_workspace_bytes(void) { return kNormCtas * (int64_t)sizeof(double); }

int ob200_launch_grad_norm(const ob200_train_tensor* tensors, int32_t n_tensors, int32_t grad_dtype, float max_norm, void* workspace,
                           float* out, ob200_stream stream) {
    const char* who = "ob200_launch_grad_norm";
    if (int rc = check_list(who, tensors, n_tensors)) return rc;
    if (!is_dtype(grad_dtype)) return set_error(OB200_ERR_INVALID, "%s: bad grad_dtype %d", who, grad_dtype);
    if (!(max_norm > 0.f)) return set_error(OB200_ERR_INVALID, "%s: max_norm has to be above 0 (infinity: no clipping)", who);
    if (!workspace || !out || (uintptr_t)workspace % 8 || (uintptr_t)out % 4)
        return set_error(OB200_ERR_INVALID, "%s: workspace or out is null or not aligned", who);
    if (n_tensors > kNormCtas * kSmallTable)
        return set_error(OB200_ERR_TOO_LARGE, "%s: more than %d tensors", who, kNormCtas * kSmallTable);
    for (int i = 0; i < n_tensors; ++i)
        if ((uintptr_t)tensors[i].grad % elem_bytes(grad_dtype)) return set_error(OB200_ERR_INVALID, "%s: tensor %d is not aligned", who, i);
    if (int rc = require_device()) return rc;
    cudaStream_t st = as_stream(stream);
    double* part = (double*)workspace;
    int parts = 0, rc;
    const bool small = n_tensors <= kSmallTable;
    if (grad_dtype == OB200_DTYPE_BF16)
        rc = small ? norm_launches<__nv_bfloat16, kSmallTable>(tensors, n_tensors, part, &parts, st) : norm_launches<__nv_bfloat16, kLargeTable>(tensors, n_tensors, part, &parts, st);
    else if (grad_dtype == OB200_DTYPE_F16)
        rc = small ? norm_launches<__half, kSmallTable>(tensors, n_tensors, part, &parts, st) : norm_launches<__half, kLargeTable>(tensors, n_tensors, part, &parts, st);
    else
        rc = small ? norm_launches<float, kSmallTable>(tensors, n_tensors, part, &parts, st) : norm_launches<float, kLargeTable>(tensors, n_tensors, part, &parts, st);
    if (rc) return rc;
    grad_norm_finish_kernel<<<1, 256, 0, st>>>(part, parts, max_norm, out);
    OB200_LAUNCHED("grad_norm_finish_kernel");
    return OB200_OK;
}

int ob200_launch_adamw(const ob200_train_tensor* tensors, int32_t n_tensors, const ob200_adamw_config* c, ob200_stream stream) {
    const char* who = "ob200_launch_adamw";
    if (!c) return set_error(OB200_ERR_INVALID, "%s: null argument", who);
    if (int rc = check_list(who, tensors, n_tensors)) return rc;
    if (!is_dtype(c->param_dtype) || !is_dtype(c->grad_dtype)) return set_error(OB200_ERR_INVALID, "%s: bad dtype", who);
    if (c->state_bits != 8 && c->state_bits != 32) return set_error(OB200_ERR_INVALID, "%s: state_bits is 8 or 32, got %d", who, c->state_bits);
    if (!(c->beta1 >= 0.0 && c->beta1 < 1.0 && c->beta2 >= 0.0 && c->beta2 < 1.0 && c->eps >= 0.0))
        return set_error(OB200_ERR_INVALID, "%s: beta1 and beta2 are in [0, 1), eps is not negative", who);
    if (!c->step_device && c->step < 1) return set_error(OB200_ERR_INVALID, "%s: step counts from 1, got %d", who, c->step);
    if (((uintptr_t)c->grad_scale | (uintptr_t)c->lr_device | (uintptr_t)c->step_device) % 4)
        return set_error(OB200_ERR_INVALID, "%s: grad_scale, lr_device or step_device is not aligned", who);
    const int pe = elem_bytes(c->param_dtype), ge = elem_bytes(c->grad_dtype), se = c->state_bits == 32 ? 4 : 1;
    for (int i = 0; i < n_tensors; ++i) {
        const ob200_train_tensor& t = tensors[i];
        if (!t.numel) continue;
        if (!t.param || !t.exp_avg || !t.exp_avg_sq || (se == 1 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
            return set_error(OB200_ERR_INVALID, "%s: tensor %d lacks its param or a state", who, i);
        if (t.exp_avg == t.exp_avg_sq) return set_error(OB200_ERR_INVALID, "%s: tensor %d has one memory for both states", who, i);
        if ((uintptr_t)t.param % pe || (uintptr_t)t.grad % ge || ((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) % se ||
            (se == 1 && ((uintptr_t)t.exp_avg_scale | (uintptr_t)t.exp_avg_sq_scale) % 4))
            return set_error(OB200_ERR_INVALID, "%s: tensor %d is not aligned", who, i);
    }
    if (int rc = check_apart(who, tensors, n_tensors, pe, &ob200_train_tensor::param, "param")) return rc;
    if (int rc = check_apart(who, tensors, n_tensors, se, &ob200_train_tensor::exp_avg, "exp_avg")) return rc;
    if (int rc = check_apart(who, tensors, n_tensors, se, &ob200_train_tensor::exp_avg_sq, "exp_avg_sq")) return rc;
    if (int rc = require_device()) return rc;
    Step k{};
    const double b1 = c->beta1, b2 = c->beta2;
    k.lr = (float)c->lr; k.beta1 = (float)b1; k.beta2 = (float)b2; k.eps = (float)c->eps;
    k.one_beta1 = (float)(1.0 - b1); k.one_beta2 = (float)(1.0 - b2);
    k.beta1_d = b1; k.beta2_d = b2;
    if (!c->step_device) {
        k.rate = (float)(1.0 / (1.0 - std::pow(b1, (double)c->step)));
        k.root = (float)(1.0 / std::sqrt(1.0 - std::pow(b2, (double)c->step)));
    }
    k.grad_scale = c->grad_scale; k.lr_device = c->lr_device; k.step_device = c->step_device;
    cudaStream_t st = as_stream(stream);
    if (c->param_dtype == OB200_DTYPE_BF16) return adamw_param<__nv_bfloat16>(tensors, n_tensors, c, k, st);
    if (c->param_dtype == OB200_DTYPE_F16) return adamw_param<__half>(tensors, n_tensors, c, k, st);
    return adamw_param<float>(tensors, n_tensors, c, k, st);
}

}  // extern "C"

// The weight update: the 2-norm of all gradients of a network with the factor that clips it, and one AdamW step over all
// its tensors, states in fp32 or in e4m3 with a scale per 256 elements.
//
// Both go over the tensors in chunks, a CTA each at a time; the list of tensors travels as a kernel parameter (up to
// 32 KB), so that a call needs no device table, no copy and no memory of its own and can be captured.  Both are bound by
// memory: every gradient, weight and state is read once and written once.
#include "common.h"
#include "packed_f32.cuh"
#include <algorithm>
#include <cmath>
#include <cstddef>
#include <memory>
#include <new>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ob200 {
namespace {

constexpr int kBlock = 256;              // elements that share the scales of 8-bit states
// Threads and elements of a CTA of AdamW: a warp takes a block, or two where the states are codes - what a warp costs besides
// its elements is a fifth of the instructions with one - and CTAs are small there, so that 28 warps fit an SM (24.5 M fp32
// weights: 63 us, with CTAs of eight warps 67, 5.5 TB/s).
template <int BITS> constexpr int kThreads = BITS == 8 ? 128 : 256;
template <int BITS> constexpr int kChunk = 2048;
template <typename G> constexpr int kNormChunk = 1024 * (16 / (int)sizeof(G));    // of a CTA's turn of the norm: 64 bytes a thread
                                         // (24.5 M bf16, 4.2 M fp32: 14.2, 6.5 us; 32 bytes 13.9, 7.2; 128 and half the CTAs 15.8, 6.5)
constexpr float kE4m3Max = 448.f, kE4m3Least = 0x1p-9f, kScaleFloor = 0x1p-110f;
constexpr int kNormCtas = 1184;          // partial sums of the norm: eight CTAs per SM

struct Entry {
    void* p; const void* g; void* m; void* v;
    float *ms, *vs;
    long long n;
    float decay;
    int vec;                             // whether four adjacent elements may be moved at once
};
// chunk0[i]: the first chunk of tensor i within the launch, rising (tensors without elements are not listed).
template <int N> struct Table { int count, chunks; int chunk0[N]; Entry e[N]; };
constexpr int kSmallTable = 48, kMiddleTable = 160, kLargeTable = 450;
static_assert(sizeof(Table<kLargeTable>) + 128 <= 32764, "the table has to fit the kernel parameters");

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// The tensor that holds a chunk.  (Lanes that count the places behind theirs read parameter memory one after the other:
// AdamW over 130 tensors took 125 us that way, 92 us with steps that all lanes take together.)
template <int N>
__device__ __forceinline__ int entry_of(const Table<N>& t, int chunk) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.chunk0[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Four adjacent elements as fp32, and back.
__device__ __forceinline__ void load4(const float* p, float* v) {
    const float4 q = *(const float4*)p;
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float* v) {
    const uint2 q = *(const uint2*)p;
    v[0] = __uint_as_float(q.x << 16); v[1] = __uint_as_float(q.x & 0xFFFF0000u);
    v[2] = __uint_as_float(q.y << 16); v[3] = __uint_as_float(q.y & 0xFFFF0000u);
}
__device__ __forceinline__ void load4(const __half* p, float* v) {
    const uint2 q = *(const uint2*)p;
    const float2 a = __half22float2(*(const __half2*)&q.x), b = __half22float2(*(const __half2*)&q.y);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
// 16 bytes of T as fp32.
__device__ __forceinline__ void load16(const float* p, float* v) { load4(p, v); }
__device__ __forceinline__ void load16(const __nv_bfloat16* p, float* v) {
    const uint4 q = *(const uint4*)p;
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}
__device__ __forceinline__ void load16(const __half* p, float* v) {
    const uint4 q = *(const uint4*)p;
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*(const __half2*)&w[i]);
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void store4(float* p, const float* v) { *(float4*)p = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *(uint2*)p = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
}
__device__ __forceinline__ void store4(__half* p, const float* v) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *(uint2*)p = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
}

// ---- norm ----------------------------------------------------------------------
// Sum of a thread's value over the CTA of eight warps, in thread 0.
__device__ __forceinline__ double cta_sum(double v) {
    __shared__ double warp_sum[8];
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = v;
    __syncthreads();
    double a = 0.0;
    if (threadIdx.x == 0)
        for (int w = 0; w < 8; ++w) a += warp_sum[w];
    return a;
}

// Squares and a thread's sums over a chunk (16 or 32 elements) in fp32, everything beyond in fp64.  The CTA that ends last
// adds up what the others left, in their order, and sets the counter back for the next call; a list that takes several
// launches is added up by the last of them.
struct NormEnd { float max_norm; float* out; unsigned* ended; int parts; };      // out null: not the last launch; parts ahead of this launch's
template <typename G, int N>
__global__ void __launch_bounds__(256)
grad_norm_kernel(const __grid_constant__ Table<N> t, double* part, const NormEnd end) {
    constexpr int V = 16 / sizeof(G);
    double sum = 0.0;
    int c = (int)((long long)t.chunks * blockIdx.x / gridDim.x);
    const int behind = (int)((long long)t.chunks * (blockIdx.x + 1) / gridDim.x);
    for (int i = entry_of(t, c); c < behind; ++c) {
        while (i + 1 < t.count && t.chunk0[i + 1] <= c) ++i;
        const Entry& e = t.e[i];
        const long long at = (long long)(c - t.chunk0[i]) * kNormChunk<G>;
        const G* g = (const G*)e.g + at;
        const int left = (int)min((long long)kNormChunk<G>, e.n - at);
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        if (e.vec && left == kNormChunk<G>) {
            float v[4][V];
#pragma unroll
            for (int i = 0; i < 4; ++i) load16(g + V * (threadIdx.x + 256 * i), v[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) s[k % 4] = fmaf(v[i][k], v[i][k], s[k % 4]);
        } else {
#pragma unroll 4
            for (int i = threadIdx.x; i < left; i += 256) {
                const float v = to_f32(g[i]);
                s[0] = fmaf(v, v, s[0]);
            }
        }
        sum += (double)((s[0] + s[1]) + (s[2] + s[3]));
    }
    sum = cta_sum(sum);
    __shared__ int last;
    if (threadIdx.x == 0) {
        part[end.parts + blockIdx.x] = sum;
        __threadfence();
        last = end.out && atomicInc(end.ended, gridDim.x - 1) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    sum = 0.0;
    for (int i = threadIdx.x; i < end.parts + (int)gridDim.x; i += 256) sum += __ldcg(part + i);
    sum = cta_sum(sum);
    if (threadIdx.x) return;
    const double norm = sqrt(sum);
    end.out[0] = (float)norm;
    // an infinite norm gives NaN, not 0: the step is to be left out, not made with zeroed gradients
    end.out[1] = !isfinite((float)norm) ? __int_as_float(0x7fc00000) : norm > (double)end.max_norm ? (float)((double)end.max_norm / norm) : 1.f;
}

// ---- AdamW ----------------------------------------------------------------------
struct Step {
    float lr, beta1, one_beta1, beta2, one_beta2, eps;
    float rate;                          // 1 / (1 - beta1^step)
    float root;                          // 1 / sqrt(1 - beta2^step)
    float one;                           // 1
    double beta1_d, beta2_d;
    const float* grad_scale; const float* lr_device; const int32_t* step_device;
};

// Two codes to two fp32 (exact), and two fp32 to two codes.
__device__ __forceinline__ void decode2(uint32_t codes, float& a, float& b) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
    const float2 f = __half22float2(*(const __half2*)&h);
    a = f.x; b = f.y;
}
__device__ __forceinline__ uint32_t encode2(float a, float b) {
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(b), "f"(a));
    return c;
}

// Largest of the warp's non-negative values (NaN is larger than all).
__device__ __forceinline__ float warp_max(float v) { return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(v))); }
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float larger(float a, float b) { return max_nan(a, fabsf(b)); }

__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A warp per block of 256, NB blocks a warp: a lane has elements 4 lane + {0..3} and 128 + 4 lane + {0..3}, or, where a
// tensor's start does not allow four at once and in its last block, lane + 32 i.
// Every product and sum of the moments is rounded by itself, as elementary operations on whole tensors round them: the codes of
// 8-bit states are a function of the inputs alone, and the one that those operations give.  Packed products and sums the
// compiler would contract, so a sum is fma(x, one, y) with a `one` that it cannot see (24.5 M weights with the
// norm: 83.6 us, as with fused sums).
template <typename P, typename G, int BITS, int N>
__global__ void __launch_bounds__(kThreads<BITS>, BITS == 8 ? 7 : 1)
adamw_kernel(const __grid_constant__ Table<N> t, const __grid_constant__ Step k) {
    constexpr int NB = kChunk<BITS> / (kThreads<BITS> / 32 * kBlock);
    const int at_entry = entry_of(t, blockIdx.x);
    const Entry& e = t.e[at_entry];
    const int lane = threadIdx.x % 32;
    const long long first = ((long long)((int)blockIdx.x - t.chunk0[at_entry]) * (kThreads<BITS> / 32) + threadIdx.x / 32) * NB;
    asm volatile("griddepcontrol.wait;" ::: "memory");       // until here nothing but the parameters was read
    const float gs = k.grad_scale ? *k.grad_scale : 1.f;
    if (!isfinite(gs) || first * kBlock >= e.n) return;
    const float lr = k.lr_device ? *k.lr_device : k.lr;
    float rate = k.rate, root = k.root;
    if (k.step_device) {
        const int32_t at = *k.step_device;
        if (at < 1) return;                  // as the host's count is refused
        const double step = (double)at;
        rate = (float)(1.0 / (1.0 - pow(k.beta1_d, step)));
        root = (float)(1.0 / sqrt(1.0 - pow(k.beta2_d, step)));
    }
    rate *= lr;
    float pe[NB][8], ge[NB][8], m[NB][8], v[NB][8], ms[NB], vs[NB];
    uint32_t mc[NB][2], vc[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const long long at = (first + b) * kBlock;
        const int left = (int)max(0LL, min((long long)kBlock, e.n - at));
        const P* p = (const P*)e.p + at;
        const G* g = (const G*)e.g + at;
        const float *m32 = (const float*)e.m + at, *v32 = (const float*)e.v + at;
        const uint8_t *m8 = (const uint8_t*)e.m + at, *v8 = (const uint8_t*)e.v + at;
        if (e.vec && left == kBlock) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = 128 * h + 4 * lane;
                load4(p + j, pe[b] + 4 * h);
                load4(g + j, ge[b] + 4 * h);
                if (BITS == 32) { load4(m32 + j, m[b] + 4 * h); load4(v32 + j, v[b] + 4 * h); }
                else { mc[b][h] = *(const uint32_t*)(m8 + j); vc[b][h] = *(const uint32_t*)(v8 + j); }
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) mc[b][h] = vc[b][h] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = lane + 32 * i;
                const bool is = j < left;
                pe[b][i] = is ? to_f32(p[j]) : 0.f;
                ge[b][i] = is ? to_f32(g[j]) : 0.f;
                if (BITS == 32) { m[b][i] = is ? m32[j] : 0.f; v[b][i] = is ? v32[j] : 0.f; }
                else if (is) { mc[b][i / 4] |= (uint32_t)m8[j] << (8 * (i % 4)); vc[b][i / 4] |= (uint32_t)v8[j] << (8 * (i % 4)); }
            }
        }
        if (BITS == 8 && left > 0) { ms[b] = e.ms[first + b]; vs[b] = e.vs[first + b]; }
    }
    const f32x2 gs2 = pair(gs, gs), b1 = pair(k.beta1, k.beta1), ob1 = pair(k.one_beta1, k.one_beta1), b2 = pair(k.beta2, k.beta2),
                ob2 = pair(k.one_beta2, k.one_beta2), root2 = pair(root, root), one2 = pair(k.one, k.one), eps2 = pair(k.eps, k.eps), rate2 = pair(-rate, -rate);
    const float keep = fmaf(-lr, e.decay, 1.f);
    const f32x2 keep2 = pair(keep, keep);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const long long at = (first + b) * kBlock;
        const int left = (int)max(0LL, min((long long)kBlock, e.n - at));
        if (left == 0) break;
        float r[8], m_top = 0.f, r_top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            f32x2 m2, v2;
            if (BITS == 32) {
                m2 = pair(m[b][i], m[b][i + 1]);
                v2 = pair(v[b][i], v[b][i + 1]);
            } else {
                float x, y;
                decode2(mc[b][i / 4] >> (8 * (i % 4)), x, y);
                m2 = mul2(pair(x, y), pair(ms[b], ms[b]));
                decode2(vc[b][i / 4] >> (8 * (i % 4)), x, y);
                v2 = mul2(pair(x, y), pair(vs[b], vs[b]));
                v2 = mul2(v2, v2);
            }
            const f32x2 g2 = mul2(pair(ge[b][i], ge[b][i + 1]), gs2);
            m2 = fma2(mul2(m2, b1), one2, mul2(g2, ob1));
            v2 = fma2(mul2(v2, b2), one2, mul2(mul2(g2, g2), ob2));
            float x, y;
            halves(v2, v[b][i], v[b][i + 1]);
            halves(m2, m[b][i], m[b][i + 1]);
            r[i] = __fsqrt_rn(v[b][i]);
            r[i + 1] = __fsqrt_rn(v[b][i + 1]);
            halves(fma2(pair(r[i], r[i + 1]), root2, eps2), x, y);
            halves(fma2(rate2, mul2(m2, pair(rcp(x), rcp(y))), mul2(pair(pe[b][i], pe[b][i + 1]), keep2)), pe[b][i], pe[b][i + 1]);
            if (BITS == 8) {
                m_top = larger(larger(m_top, m[b][i]), m[b][i + 1]);
                r_top = larger(larger(r_top, r[i]), r[i + 1]);
            }
        }
        P* p = (P*)e.p + at;
        float *m32 = (float*)e.m + at, *v32 = (float*)e.v + at;
        uint8_t *m8 = (uint8_t*)e.m + at, *v8 = (uint8_t*)e.v + at;
        const bool vec = e.vec && left == kBlock;
        if (vec) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = 128 * h + 4 * lane;
                store4(p + j, pe[b] + 4 * h);
                if (BITS == 32) { store4(m32 + j, m[b] + 4 * h); store4(v32 + j, v[b] + 4 * h); }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = lane + 32 * i;
                if (j >= left) continue;
                p[j] = from_f32<P>(pe[b][i]);
                if (BITS == 32) { m32[j] = m[b][i]; v32[j] = v[b][i]; }
            }
        }
        if (BITS == 32) continue;
        m_top = warp_max(m_top); r_top = warp_max(r_top);
        if (m_top < kScaleFloor) m_top = kScaleFloor;
        if (r_top < kScaleFloor) r_top = kScaleFloor;
        // both reciprocals in one, a lane each
        const float top = lane & 1 ? r_top : m_top, ratio = __fmul_rn(__frcp_rn(top), kE4m3Max);
        const float mi = __shfl_sync(~0u, ratio, 0), ri = __shfl_sync(~0u, ratio, 1);
        // an infinite maximum's scale is NaN, else a root above 0 would be infinite and its weight stand still
        if (lane < 2) (lane ? e.vs : e.ms)[first + b] = __fmul_rn(top + (top - top), 1.f / kE4m3Max);
        const f32x2 mi2 = pair(mi, mi), ri2 = pair(ri, ri);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t c[4];
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                float x, y;
                halves(mul2(pair(m[b][4 * h + i], m[b][4 * h + i + 1]), mi2), x, y);
                c[i] = encode2(x, y);
                halves(mul2(pair(r[4 * h + i], r[4 * h + i + 1]), ri2), x, y);
                if (r[4 * h + i] > 0.f) x = max_nan(x, kE4m3Least);
                if (r[4 * h + i + 1] > 0.f) y = max_nan(y, kE4m3Least);
                c[i + 1] = encode2(x, y);
            }
            mc[b][h] = __byte_perm(c[0], c[2], 0x5410);
            vc[b][h] = __byte_perm(c[1], c[3], 0x5410);
        }
        if (vec) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = 128 * h + 4 * lane;
                *(uint32_t*)(m8 + j) = mc[b][h];
                *(uint32_t*)(v8 + j) = vc[b][h];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = lane + 32 * i;
                if (j >= left) continue;
                m8[j] = (uint8_t)(mc[b][i / 4] >> (8 * (i % 4)));
                v8[j] = (uint8_t)(vc[b][i / 4] >> (8 * (i % 4)));
            }
        }
    }
}

// ---- host ----------------------------------------------------------------------
int elem_bytes(int dtype) { return dtype == OB200_DTYPE_F32 ? 4 : 2; }
bool is_dtype(int d) { return d == OB200_DTYPE_BF16 || d == OB200_DTYPE_F16 || d == OB200_DTYPE_F32; }

// Fills t with tensors [*next, n) as far as they fit; false when there was nothing left to take.
// chunk: elements; wide: bytes that p, g and the states have to be aligned to for four elements at once, 1 where it does not matter.
struct Wide { uintptr_t p, g, state; };
template <int N>
bool fill_table(Table<N>* t, const ob200_train_tensor* in, int n, int chunk, Wide wide, int* next, long long* chunks) {
    t->count = 0;
    *chunks = 0;
    for (; *next < n && t->count < N; ++*next) {
        const ob200_train_tensor& a = in[*next];
        if (a.numel == 0) continue;
        const long long c = (a.numel + chunk - 1) / chunk;
        if (t->count && *chunks + c > 0x7fffffffLL) break;   // the rest in another launch
        t->chunk0[t->count] = (int)*chunks;
        t->e[t->count++] = Entry{a.param, a.grad, a.exp_avg, a.exp_avg_sq, a.exp_avg_scale, a.exp_avg_sq_scale, a.numel, a.weight_decay,
                               (((uintptr_t)a.param & (wide.p - 1)) | ((uintptr_t)a.grad & (wide.g - 1)) | (((uintptr_t)a.exp_avg | (uintptr_t)a.exp_avg_sq) & (wide.state - 1))) == 0};
        *chunks += c;
    }
    t->chunks = (int)*chunks;
    return t->count > 0;
}

constexpr long long kMostElements = 0x7fffffffLL * 2048;

int check_list(const char* who, const ob200_train_tensor* t, int n) {
    if (n < 0 || (n > 0 && !t)) return set_error(OB200_ERR_INVALID, "%s: null tensors or a negative count", who);
    for (int i = 0; i < n; ++i) {
        if (t[i].numel < 0) return set_error(OB200_ERR_INVALID, "%s: tensor %d has a negative size", who, i);
        if (t[i].numel > kMostElements) return set_error(OB200_ERR_TOO_LARGE, "%s: tensor %d has too many elements", who, i);
        if (t[i].numel && !t[i].grad) return set_error(OB200_ERR_INVALID, "%s: tensor %d has no gradient", who, i);
    }
    return OB200_OK;
}

template <typename G, int N>
int norm_launches(const ob200_train_tensor* tensors, int n, double* part, float max_norm, float* out, cudaStream_t st) {
    Table<N> t;
    int next = 0, parts = 0;
    long long chunks;
    do {
        fill_table(&t, tensors, n, kNormChunk<G>, Wide{1, 16, 1}, &next, &chunks);
        // lists of more than one launch share the places of partial sums out
        const int room = kNormCtas - parts, more = (n - next + N - 1) / N;
        if (room < 1) return set_error(OB200_ERR_TOO_LARGE, "ob200_launch_grad_norm: too many tensors");
        const int ctas = (int)std::max(1LL, std::min<long long>(chunks, std::max(1, room / (1 + more))));
        const NormEnd end{max_norm, next == n ? out : nullptr, (unsigned*)(part + kNormCtas), parts};
        grad_norm_kernel<G, N><<<ctas, 256, 0, st>>>(t, part, end);
        OB200_LAUNCHED("grad_norm_kernel");
        parts += ctas;
    } while (next < n);
    return OB200_OK;
}

template <typename G>
int norm_typed(const ob200_train_tensor* tensors, int n, double* part, float max_norm, float* out, cudaStream_t st) {
    if (n <= kSmallTable) return norm_launches<G, kSmallTable>(tensors, n, part, max_norm, out, st);
    return n <= kMiddleTable ? norm_launches<G, kMiddleTable>(tensors, n, part, max_norm, out, st) : norm_launches<G, kLargeTable>(tensors, n, part, max_norm, out, st);
}

template <typename P, typename G, int BITS, int N>
int adamw_launches(const ob200_train_tensor* tensors, int n, const Step& k, cudaStream_t st) {
    Table<N> t;
    int next = 0;
    long long chunks;
    while (fill_table(&t, tensors, n, kChunk<BITS>, Wide{4 * sizeof(P), 4 * sizeof(G), BITS == 32 ? 16 : 4}, &next, &chunks)) {
        OB200_CUDA_OK(launch_dependent(adamw_kernel<P, G, BITS, N>, dim3((unsigned)chunks), dim3(kThreads<BITS>), 0, st, t, k));
        OB200_LAUNCHED("adamw_kernel");
    }
    return OB200_OK;
}

template <typename P, typename G>
int adamw_typed(const ob200_train_tensor* tensors, int n, int bits, const Step& k, cudaStream_t st) {
    if (n <= kSmallTable)
        return bits == 8 ? adamw_launches<P, G, 8, kSmallTable>(tensors, n, k, st) : adamw_launches<P, G, 32, kSmallTable>(tensors, n, k, st);
    if (n <= kMiddleTable)
        return bits == 8 ? adamw_launches<P, G, 8, kMiddleTable>(tensors, n, k, st) : adamw_launches<P, G, 32, kMiddleTable>(tensors, n, k, st);
    return bits == 8 ? adamw_launches<P, G, 8, kLargeTable>(tensors, n, k, st) : adamw_launches<P, G, 32, kLargeTable>(tensors, n, k, st);
}

template <typename P>
int adamw_param(const ob200_train_tensor* tensors, int n, const ob200_adamw_config* c, const Step& k, cudaStream_t st) {
    if (c->grad_dtype == OB200_DTYPE_BF16) return adamw_typed<P, __nv_bfloat16>(tensors, n, c->state_bits, k, st);
    if (c->grad_dtype == OB200_DTYPE_F16) return adamw_typed<P, __half>(tensors, n, c->state_bits, k, st);
    return adamw_typed<P, float>(tensors, n, c->state_bits, k, st);
}

// Memory of one kind that a call writes: `bytes` for every 2^shift elements of a tensor (scales: a float for 256).
struct Written { const char* what; size_t at; int bytes, shift; };       // at: the pointer's place in an ob200_train_tensor
// Whether two tensors of a call share memory that it writes: two CTAs would update it at once.
int check_apart(const char* who, const ob200_train_tensor* t, int n, const Written* kinds, int n_kinds) {
    auto begin = [&](const Written& k, int i) {
        uintptr_t at;
        std::memcpy(&at, (const char*)(t + i) + k.at, sizeof(at));
        return at;
    };
    auto end = [&](const Written& k, int i) { return begin(k, i) + (uintptr_t)((t[i].numel + (1 << k.shift) - 1) >> k.shift) * k.bytes; };
    // in the order of memory, as the views of flat buffers are, each kind in a buffer of its own
    uintptr_t lo[5], hi[5];
    bool apart = true;
    for (int k = 0; k < n_kinds && apart; ++k) {
        const Written kind = kinds[k];
        uintptr_t first = 0, last = 0;
        for (int i = 0; i < n && apart; ++i) {
            if (!t[i].numel) continue;
            const uintptr_t at = begin(kind, i);
            if (!last) first = at;
            else apart = at >= last;
            last = end(kind, i);
        }
        lo[k] = first; hi[k] = last;
        for (int q = 0; q < k && apart; ++q) apart = hi[k] <= lo[q] || hi[q] <= lo[k];
    }
    if (apart) return OB200_OK;
    struct Span { uintptr_t begin, end; int kind, i; };
    std::unique_ptr<Span[]> all(new (std::nothrow) Span[(size_t)n * n_kinds]);
    if (!all) return set_error(OB200_ERR_STATE, "%s: out of host memory", who);
    size_t count = 0;
    for (int k = 0; k < n_kinds; ++k)
        for (int i = 0; i < n; ++i)
            if (t[i].numel) all[count++] = Span{begin(kinds[k], i), end(kinds[k], i), k, i};
    std::sort(all.get(), all.get() + count, [](const Span& a, const Span& b) { return a.begin < b.begin; });
    for (size_t s = 1; s < count; ++s)
        if (all[s].begin < all[s - 1].end)
            return set_error(OB200_ERR_INVALID, "%s: %s of tensor %d and %s of tensor %d share memory", who, kinds[all[s - 1].kind].what,
                             all[s - 1].i, kinds[all[s].kind].what, all[s].i);
    return OB200_OK;
}

}  // namespace
}  // namespace ob200

using namespace ob200;

extern "C" {

int64_t ob200_grad_norm_workspace_bytes(void) { return (kNormCtas + 1) * (int64_t)sizeof(double); }

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
    if (grad_dtype == OB200_DTYPE_BF16) return norm_typed<__nv_bfloat16>(tensors, n_tensors, part, max_norm, out, st);
    if (grad_dtype == OB200_DTYPE_F16) return norm_typed<__half>(tensors, n_tensors, part, max_norm, out, st);
    return norm_typed<float>(tensors, n_tensors, part, max_norm, out, st);
}

int ob200_launch_adamw(const ob200_train_tensor* tensors, int32_t n_tensors, const ob200_adamw_config* c, ob200_stream stream) {
    const char* who = "ob200_launch_adamw";
    if (!c) return set_error(OB200_ERR_INVALID, "%s: null argument", who);
    if (int rc = check_list(who, tensors, n_tensors)) return rc;
    if (!is_dtype(c->param_dtype) || !is_dtype(c->grad_dtype)) return set_error(OB200_ERR_INVALID, "%s: bad dtype", who);
    if (c->state_bits != 8 && c->state_bits != 32) return set_error(OB200_ERR_INVALID, "%s: state_bits is 8 or 32, got %d", who, c->state_bits);
    if (!(c->beta1 >= 0.0 && c->beta1 < 1.0 && c->beta2 >= 0.0 && c->beta2 < 1.0 && c->eps >= 0.0))
        return set_error(OB200_ERR_INVALID, "%s: beta1 and beta2 are in [0, 1), eps is not negative", who);
    if ((float)c->eps > 0.f && (float)c->eps < 0x1p-126f)        // the reciprocal of a subnormal sum is infinite, times a moment of 0 NaN
        return set_error(OB200_ERR_INVALID, "%s: eps is 0 or at least 2^-126 in fp32", who);
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
    using Tensor = ob200_train_tensor;
    const Written kinds[5] = {{"param", offsetof(Tensor, param), pe, 0}, {"exp_avg", offsetof(Tensor, exp_avg), se, 0},
                              {"exp_avg_sq", offsetof(Tensor, exp_avg_sq), se, 0}, {"exp_avg_scale", offsetof(Tensor, exp_avg_scale), 4, 8},
                              {"exp_avg_sq_scale", offsetof(Tensor, exp_avg_sq_scale), 4, 8}};
    static_assert(kBlock == 1 << 8, "a scale's elements");
    if (int rc = check_apart(who, tensors, n_tensors, kinds, se == 1 ? 5 : 3)) return rc;
    if (int rc = require_device()) return rc;
    Step k{};
    const double b1 = c->beta1, b2 = c->beta2;
    k.lr = (float)c->lr; k.beta1 = (float)b1; k.beta2 = (float)b2; k.eps = (float)c->eps;
    k.one = 1.f;
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

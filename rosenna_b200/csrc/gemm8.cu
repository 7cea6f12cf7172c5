// The 8-bit Gemm (gemm8.cuh).
//
// Scales are powers of two: a block's is 2^e with the least e >= -126 for which
// its largest magnitude is at most 448 * 2^e (448: the largest e4m3 value), so
// dividing by it is exact and each value is rounded once, to nearest even.  A
// column whose block holds an infinity or NaN gives NaN.
#include "gemm8.cuh"

#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <cstring>

namespace rosenna {
namespace {

constexpr int kThreads = 256;

// exponent of the scale of a block with largest magnitude `bits` (the bits of a
// positive finite float): 448 = 1.75 * 2^8
__host__ __device__ __forceinline__ int block_exponent(uint32_t bits) {
    if (bits == 0) return 0;
    const int q = (int)(bits >> 23) - 127;
    const int e = q - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}

// nearest e4m3 (ties to even) of a finite v, |v| <= 448
uint8_t to_e4m3(float v) {
    const uint8_t sign = std::signbit(v) ? 0x80 : 0;
    const double a = std::fabs((double)v);
    if (a == 0.0) return sign;
    const int e = std::max(std::ilogb(a), -6);
    const int m = (int)std::nearbyint(std::ldexp(a, 3 - e));  // in eighths of 2^e; 16 carries into the exponent
    return (uint8_t)(sign | (((e + 6) << 3) + m));
}

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float apply_act(float v, int act) {
    switch (act) {
        case 1: return v < 0.f ? 0.f : v;
        case 2: return 1.f - __fdividef(2.f, 1.f + ex2_approx(2.8853900817779268f * v));
        case 3: return __fdividef(1.f, 1.f + ex2_approx(-1.4426950408889634f * v));
        case 4: return __fdividef(v, 1.f + ex2_approx(-1.4426950408889634f * v));
        default: return v;
    }
}

// four values, already divided by the scale, as e4m3 bytes (lowest first)
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// One thread per (column, block of 128 rows).
__global__ void __launch_bounds__(kThreads) gemm8_quantise_kernel(const Gemm8Args p) {
    const long long c = (long long)blockIdx.x * kThreads + threadIdx.x;
    const int kb = blockIdx.y;
    if (c >= p.n) return;
    const float *x = p.x + (long long)kb * kGemm8Block * p.ld_x + c;
    const int rows = min(kGemm8Block, p.K - kb * kGemm8Block);
    uint32_t amax = 0;
    for (int k = 0; k < rows; k++) amax = max(amax, __float_as_uint(x[k * p.ld_x]) & 0x7fffffffu);
    const bool finite = amax < 0x7f800000u;
    const int e = finite ? block_exponent(amax) : 0;
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    p.xs[(long long)kb * p.n + c] = finite ? __uint_as_float((uint32_t)(127 + e) << 23) : __uint_as_float(0x7fc00000u);
    uint4 *out = reinterpret_cast<uint4 *>(p.xq + c * p.Kp + kb * kGemm8Block);
    for (int k = 0; k < kGemm8Block; k += 16) {
        uint32_t v[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            float f[4];
#pragma unroll
            for (int r = 0; r < 4; r++) f[r] = k + 4 * q + r < rows ? x[(k + 4 * q + r) * p.ld_x] * inv : 0.f;
            v[q] = e4m3x4(f[0], f[1], f[2], f[3]);
        }
        out[k / 16] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

__device__ __forceinline__ void unpack4(uint32_t v, float (&f)[4]) {
    __nv_fp8x4_e4m3 q;
    q.__x = v;
    const float4 r = static_cast<float4>(q);
    f[0] = r.x;
    f[1] = r.y;
    f[2] = r.z;
    f[3] = r.w;
}

// One thread per column and 8 outputs.
__global__ void __launch_bounds__(kThreads) gemm8_simple_kernel(const Gemm8Args p) {
    const long long c = (long long)blockIdx.x * kThreads + threadIdx.x;
    const int m0 = blockIdx.y * 8;
    if (c >= p.n) return;
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = 0.f;
    const int nkb = p.Kp / kGemm8Block;
    for (int kb = 0; kb < nkb; kb++) {
        float part[8];
#pragma unroll
        for (int i = 0; i < 8; i++) part[i] = 0.f;
        for (int k = 0; k < kGemm8Block; k += 4) {
            float xf[4], wf[4];
            unpack4(*reinterpret_cast<const uint32_t *>(p.xq + c * p.Kp + kb * kGemm8Block + k), xf);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                unpack4(*reinterpret_cast<const uint32_t *>(p.wq + (long long)(m0 + i) * p.Kp + kb * kGemm8Block + k), wf);
#pragma unroll
                for (int r = 0; r < 4; r++) part[i] = fmaf(xf[r], wf[r], part[i]);
            }
        }
        const float sc = p.xs[(long long)kb * p.n + c] * p.ws[(m0 / kGemm8Block) * nkb + kb];
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] = fmaf(part[i], sc, acc[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (m0 + i < p.M) p.y[(long long)(m0 + i) * p.ld_y + c] = apply_act(acc[i] + (p.bias ? p.bias[m0 + i] : 0.f), p.act);
}

}  // namespace

void gemm8_pack(const float *w, int M, int K, Gemm8Weights *out) {
    out->M = M;
    out->K = K;
    out->Mp = (M + kGemm8Block - 1) / kGemm8Block * kGemm8Block;
    out->Kp = (K + kGemm8Block - 1) / kGemm8Block * kGemm8Block;
    const int nkb = out->Kp / kGemm8Block;
    out->q.assign((size_t)out->Mp * out->Kp, 0);
    out->scale.assign((size_t)(out->Mp / kGemm8Block) * nkb, 1.f);
    for (int mb = 0; mb < out->Mp; mb += kGemm8Block)
        for (int kb = 0; kb < out->Kp; kb += kGemm8Block) {
            float amax = 0.f;
            const int m1 = std::min(M, mb + kGemm8Block), k1 = std::min(K, kb + kGemm8Block);
            for (int m = mb; m < m1; m++)
                for (int k = kb; k < k1; k++) amax = std::max(amax, std::fabs(w[(size_t)m * K + k]));
            uint32_t bits;
            std::memcpy(&bits, &amax, 4);
            const int e = block_exponent(bits);
            out->scale[(size_t)(mb / kGemm8Block) * nkb + kb / kGemm8Block] = std::ldexp(1.f, e);
            for (int m = mb; m < m1; m++)
                for (int k = kb; k < k1; k++)
                    out->q[(size_t)m * out->Kp + k] = to_e4m3(std::ldexp(w[(size_t)m * K + k], -e));
        }
}

size_t gemm8_workspace_bytes(long long n, int M, int K) {
    (void)M;
    const size_t kp = (size_t)(K + kGemm8Block - 1) / kGemm8Block * kGemm8Block;
    return (size_t)n * kp + (size_t)n * (kp / kGemm8Block) * sizeof(float);
}

cudaError_t launch_gemm8(Gemm8Args a, void *workspace, int num_sms, cudaStream_t st, int *launches) {
    (void)num_sms;
    a.xq = static_cast<uint8_t *>(workspace);
    a.xs = reinterpret_cast<float *>(a.xq + (size_t)a.n * a.Kp);
    const unsigned cols = (unsigned)((a.n + kThreads - 1) / kThreads);
    gemm8_quantise_kernel<<<dim3(cols, (unsigned)(a.Kp / kGemm8Block)), kThreads, 0, st>>>(a);
    gemm8_simple_kernel<<<dim3(cols, (unsigned)((a.M + 7) / 8)), kThreads, 0, st>>>(a);
    *launches = 2;
    return cudaGetLastError();
}

}  // namespace rosenna

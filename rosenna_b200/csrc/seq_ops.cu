// The sequence operators of a selective state space layer: the short causal
// depthwise convolution in front of it and the selective scan itself, for whole
// histories and for single steps with the state carried by the caller.
#include "seq_ops.cuh"

#include <algorithm>

namespace rosenna {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.f + ex2_approx(-kLog2e * v)); }
// max(v, 0) + log(1 + e^-|v|): exact to a few ulp for every v, also where the
// result is tiny (log1pf), since the step length scales the whole update
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.f) + log1pf(ex2_approx(-kLog2e * fabsf(v))); }

__device__ __forceinline__ int clamp_len(const int *lens, long long s, int T) {
    return lens ? min(max(lens[s], 0), T) : T;
}

// ---- causal convolution ------------------------------------------------------
// One thread per (sample, channel, tile of kConvTile steps): a sliding window of
// W inputs in registers.
constexpr int kConvTile = 16;

template <int W>
__global__ void __launch_bounds__(kThreads) causal_conv_kernel(const CausalConvArgs p, int tiles) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= p.n * tiles * p.D) return;
    const long long s = i % p.n, r = i / p.n;
    const int tile = (int)(r % tiles), d = (int)(r / tiles);
    const int len = clamp_len(p.lens, s, p.T), t0 = tile * kConvTile, t1 = min(t0 + kConvTile, len);
    float w[W], win[W];
    win[0] = 0.f;
#pragma unroll
    for (int k = 0; k < W; k++) w[k] = p.w[d * W + k];
    const float b = p.bias ? p.bias[d] : 0.f;
    const float *x = p.x + (long long)p.T * d * p.ld_x + s;
    const float *si = p.s_in ? p.s_in + (long long)(W - 1) * d * p.ld_s_in + s : nullptr;
    // win[k] = input k - (W-1) steps after t0; the first tile's lie in the state
#pragma unroll
    for (int k = 0; k < W - 1; k++) {
        if (tile == 0) win[k + 1] = si ? si[k * p.ld_s_in] : 0.f;
        else if (t0 < t1) win[k + 1] = x[(long long)(t0 - (W - 1) + k) * p.ld_x];
    }
    if (tile == 0 && p.s_out) {
        // the new state, by the thread that alone reads the old one (they may
        // be the same array): the last W-1 of (old state, inputs before len)
        float ns[W];
#pragma unroll
        for (int k = 0; k < W - 1; k++) {
            const int t = len - (W - 1) + k;
            float v = 0.f;
            if (t >= 0) {
                v = x[(long long)t * p.ld_x];
            } else {
#pragma unroll
                for (int q = 0; q < W - 1; q++)
                    if (t + W - 1 == q) v = win[q + 1];
            }
            ns[k] = v;
        }
#pragma unroll
        for (int k = 0; k < W - 1; k++) p.s_out[((long long)(W - 1) * d + k) * p.ld_s_out + s] = ns[k];
    }
    float *y = p.y + (long long)p.T * d * p.ld_y + s;
    for (int t = t0; t < t1; t++) {
#pragma unroll
        for (int k = 0; k < W - 1; k++) win[k] = win[k + 1];
        win[W - 1] = x[(long long)t * p.ld_x];
        float v = b;
#pragma unroll
        for (int k = 0; k < W; k++) v = fmaf(w[k], win[k], v);
        y[(long long)t * p.ld_y] = p.silu ? silu(v) : v;
    }
}

// ---- selective scan --------------------------------------------------------------
// One thread per (sample, channel, chunk of time), the N states in registers.
// PASS 0: the whole length in one go.  PASS 1: a chunk from a zero state, leaving
// its final state and summed step; PASS 2: a chunk from the state it starts in.
template <int NP, int PASS>
__global__ void __launch_bounds__(kThreads) scan_kernel(const ScanArgs p) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= p.n * p.D) return;
    const long long s = i % p.n;
    const int d = (int)(i / p.n), g = d / (p.D / p.G), c = blockIdx.y;
    const int len = clamp_len(p.lens, s, p.T), t0 = c * p.chunk, t1 = min(t0 + p.chunk, len);
    float A[NP], h[NP];
#pragma unroll
    for (int j = 0; j < NP; j++) {
        A[j] = j < p.N ? p.A[(long long)d * p.N + j] * kLog2e : 0.f;
        h[j] = 0.f;
    }
    if (PASS == 0 && p.h0) {
#pragma unroll
        for (int j = 0; j < NP; j++)
            if (j < p.N) h[j] = p.h0[((long long)p.N * d + j) * p.ld_h0 + s];
    }
    if (PASS == 2) {
#pragma unroll
        for (int j = 0; j < NP; j++)
            if (j < p.N) h[j] = p.ws_h[(((long long)c * p.N + j) * p.D + d) * p.n + s];
    }
    const float bias = p.dt_bias ? p.dt_bias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
    const float *x = p.x + (long long)p.T * d * p.ld_x + s, *dt = p.dt + (long long)p.T * d * p.ld_dt + s;
    const float *z = p.z ? p.z + (long long)p.T * d * p.ld_z + s : nullptr;
    const float *B = p.B + (long long)p.T * p.N * g * p.ld_B + s, *C = p.C + (long long)p.T * p.N * g * p.ld_C + s;
    float *y = p.y + (long long)p.T * d * p.ld_y + s;
    float sum = 0.f;
    for (int t = t0; t < t1; t++) {
        float delta = dt[(long long)t * p.ld_dt] + bias;
        if (p.softplus) delta = softplus(delta);
        const float xv = x[(long long)t * p.ld_x], u = delta * xv;
        float acc = 0.f;
        sum += delta;
#pragma unroll
        for (int j = 0; j < NP; j++) {
            if (j >= p.N) break;
            const long long row = t + (long long)p.T * j;
            h[j] = fmaf(ex2_approx(delta * A[j]), h[j], u * B[row * p.ld_B]);
            if (PASS != 1) acc = fmaf(C[row * p.ld_C], h[j], acc);
        }
        if (PASS != 1) {
            acc = fmaf(skip, xv, acc);
            if (z) acc *= silu(z[(long long)t * p.ld_z]);
            y[(long long)t * p.ld_y] = acc;
        }
    }
    if (PASS == 0 && p.hn) {
#pragma unroll
        for (int j = 0; j < NP; j++)
            if (j < p.N) p.hn[((long long)p.N * d + j) * p.ld_hn + s] = h[j];
    }
    if (PASS == 1) {
#pragma unroll
        for (int j = 0; j < NP; j++)
            if (j < p.N) p.ws_h[(((long long)c * p.N + j) * p.D + d) * p.n + s] = h[j];
        p.ws_d[((long long)c * p.D + d) * p.n + s] = sum;
    }
}

// Joins the chunks: one thread per (sample, channel, state) walks them in order
// and replaces each chunk's own final state by the state it starts in.
__global__ void __launch_bounds__(kThreads) scan_carry_kernel(const ScanArgs p) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x, nd = p.n * p.D;
    if (i >= nd * p.N) return;
    const long long sd = i % nd, s = sd % p.n;
    const int j = (int)(i / nd), d = (int)(sd / p.n);
    const float A = p.A[(long long)d * p.N + j] * kLog2e;
    float h = p.h0 ? p.h0[((long long)p.N * d + j) * p.ld_h0 + s] : 0.f;
    for (int c = 0; c < p.chunks; c++) {
        float *w = p.ws_h + ((long long)c * p.N + j) * nd + sd;
        const float part = *w;
        *w = h;
        h = fmaf(ex2_approx(p.ws_d[c * nd + sd] * A), h, part);
    }
    if (p.hn) p.hn[((long long)p.N * d + j) * p.ld_hn + s] = h;
}

template <int NP>
cudaError_t launch_scan_n(const ScanArgs &a, cudaStream_t st, int *launches) {
    const long long nd = a.n * a.D;
    const unsigned blocks = (unsigned)((nd + kThreads - 1) / kThreads);
    if (a.chunks == 1) {
        scan_kernel<NP, 0><<<dim3(blocks, 1), kThreads, 0, st>>>(a);
        *launches = 1;
    } else {
        scan_kernel<NP, 1><<<dim3(blocks, (unsigned)a.chunks), kThreads, 0, st>>>(a);
        scan_carry_kernel<<<(unsigned)((nd * a.N + kThreads - 1) / kThreads), kThreads, 0, st>>>(a);
        scan_kernel<NP, 2><<<dim3(blocks, (unsigned)a.chunks), kThreads, 0, st>>>(a);
        *launches = 3;
    }
    return cudaGetLastError();
}

}  // namespace

void scan_split(long long n, int T, int D, int N, int *chunk, int *chunks) {
    (void)N;
    *chunk = std::max(T, 1);
    *chunks = 1;
    const long long want = 148LL * 1024, have = std::max(1LL, n * D);
    if (have * 2 > want || T < 64) return;
    const int c = (int)std::min<long long>((want + have - 1) / have, T / 32);
    if (c < 2) return;
    *chunk = (T + c - 1) / c;
    *chunks = (T + *chunk - 1) / *chunk;
}

size_t scan_workspace_bytes(long long n, int T, int D, int N) {
    int chunk, chunks;
    scan_split(n, T, D, N, &chunk, &chunks);
    return chunks == 1 ? 0 : sizeof(float) * (size_t)n * (size_t)D * (size_t)chunks * (size_t)(N + 1);
}

void scan_bind_workspace(ScanArgs *a, void *workspace) {
    scan_split(a->n, a->T, a->D, a->N, &a->chunk, &a->chunks);
    if (!workspace) {
        a->chunk = std::max(a->T, 1);
        a->chunks = 1;
    }
    a->ws_h = static_cast<float *>(workspace);
    a->ws_d = a->ws_h ? a->ws_h + (size_t)a->n * a->D * a->N * a->chunks : nullptr;
}

cudaError_t launch_causal_conv(const CausalConvArgs &a, cudaStream_t st) {
    const int tiles = std::max(1, (a.T + kConvTile - 1) / kConvTile);
    const unsigned blocks = (unsigned)((a.n * tiles * a.D + kThreads - 1) / kThreads);
    switch (a.W) {
        case 1: causal_conv_kernel<1><<<blocks, kThreads, 0, st>>>(a, tiles); break;
        case 2: causal_conv_kernel<2><<<blocks, kThreads, 0, st>>>(a, tiles); break;
        case 3: causal_conv_kernel<3><<<blocks, kThreads, 0, st>>>(a, tiles); break;
        case 4: causal_conv_kernel<4><<<blocks, kThreads, 0, st>>>(a, tiles); break;
        case 5: causal_conv_kernel<5><<<blocks, kThreads, 0, st>>>(a, tiles); break;
        case 6: causal_conv_kernel<6><<<blocks, kThreads, 0, st>>>(a, tiles); break;
        case 7: causal_conv_kernel<7><<<blocks, kThreads, 0, st>>>(a, tiles); break;
        case 8: causal_conv_kernel<8><<<blocks, kThreads, 0, st>>>(a, tiles); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

cudaError_t launch_scan(const ScanArgs &a, cudaStream_t st, int *launches) {
    if (a.N <= 4) return launch_scan_n<4>(a, st, launches);
    if (a.N <= 8) return launch_scan_n<8>(a, st, launches);
    if (a.N <= 16) return launch_scan_n<16>(a, st, launches);
    if (a.N <= 32) return launch_scan_n<32>(a, st, launches);
    return launch_scan_n<kMaxScanStates>(a, st, launches);
}

}  // namespace rosenna

// The sequence operators of a selective state space layer: the short causal
// depthwise convolution in front of it and the selective scan itself, for whole
// histories and for single steps with the state carried by the caller.
#include "seq_ops.cuh"

#include <algorithm>
#include <type_traits>

namespace rosenna {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float silu(float v) { return v * rcp_approx(1.f + ex2_approx(-kLog2e * v)); }
// max(v, 0) + log(1 + e), e = e^-|v| <= 1.  The step length scales the whole update,
// so the logarithm keeps its relative accuracy where e is small: log(1 + e) =
// 2 atanh(s) with s = e / (2 + e) <= 1/3, and atanh(s)/s as a polynomial in s^2 (a
// minimax fit on [0, 1/9], off by 4e-9).
__device__ __forceinline__ float softplus(float v) {
    const float e = ex2_approx(-kLog2e * fabsf(v));
    const float s = e * rcp_approx(2.f + e), w = s * s;
    float r = fmaf(0.2817831039428711f, w, 0.27960607409477234f);
    r = fmaf(r, w, 0.40024909377098083f);
    r = fmaf(r, w, 0.6666631698608398f);
    r = fmaf(r, w, 2.f);
    return fmaf(r, s, fmaxf(v, 0.f));
}

__device__ __forceinline__ int clamp_len(const int *lens, long long s, int T) {
    return lens ? min(max(lens[s], 0), T) : T;
}

// V samples next to each other (V = 4: 16-byte accesses)
template <int V>
struct Vals {
    float v[V];
};
template <int V>
__device__ __forceinline__ Vals<V> load_vals(const float *q) {
    Vals<V> r;
    if constexpr (V == 4) *reinterpret_cast<float4 *>(&r) = *reinterpret_cast<const float4 *>(q);
    else r.v[0] = *q;
    return r;
}
template <int V>
__device__ __forceinline__ void store_vals(float *q, const Vals<V> &r) {
    if constexpr (V == 4) *reinterpret_cast<float4 *>(q) = *reinterpret_cast<const float4 *>(&r);
    else *q = r.v[0];
}

// ---- causal convolution ------------------------------------------------------
// Both kernels only move data: every input is read once from memory, the taps'
// other reads of it are the registers' or L1's.  4 taps: 65536 samples x 64 channels,
// one step, 24 us (5.7 TB/s); 16384 x 50 steps x 64, 74 us (5.6 TB/s).
//
// Many samples: one thread per (V samples, run of `run` tiles of TT steps, channel),
// which keeps the last W - 1 inputs and has the next tile's loads in flight while it
// works on one.  The thread of the first run also writes the new state: it alone
// reads the old one, so the two may be the same array.
template <int W, int V, int TT>
__global__ void __launch_bounds__(kThreads, V > 1 ? 2 : 1) causal_conv_kernel(const CausalConvArgs p, int runs, int run, unsigned sample_blocks) {
    static_assert(TT >= W - 1 || TT == 1, "a tile refills the window");
    // blockDim.x threads along the samples (V = 4: n is a multiple of 4), blockDim.y
    // along (run, channel)
    const unsigned rb = blockIdx.x / sample_blocks, r = rb * blockDim.y + threadIdx.y;
    const long long s = ((long long)(blockIdx.x - rb * sample_blocks) * blockDim.x + threadIdx.x) * V;
    const int d = (int)(r / (unsigned)runs), ri = (int)(r - (unsigned)d * runs), t0 = ri * run * TT;
    if (s >= p.n || d >= p.D) return;
    int len[V], most = 0, least = p.T;
#pragma unroll
    for (int e = 0; e < V; e++) {
        len[e] = clamp_len(p.lens, s + e, p.T);
        most = max(most, len[e]);
        least = min(least, len[e]);
    }
    const bool state = ri == 0 && W > 1 && p.s_out;
    const int t1 = min(most, t0 + run * TT);
    if (t0 >= t1 && !state) return;
    float w[W];
#pragma unroll
    for (int k = 0; k < W; k++) w[k] = __ldg(p.w + d * W + k);
    const float b = p.bias ? __ldg(p.bias + d) : 0.f;
    const float *x = p.x + ((long long)p.T * d + t0) * p.ld_x + s;
    const float *si = p.s_in ? p.s_in + (long long)(W - 1) * d * p.ld_s_in + s : nullptr;
    // win[k]: the input k - (W-1) steps after the tile's first; the first run's
    // earlier ones are the state
    Vals<V> win[TT + W - 1], next[TT];
#pragma unroll
    for (int k = 0; k < W - 1; k++) {
#pragma unroll
        for (int e = 0; e < V; e++) win[k].v[e] = 0.f;
        if (ri > 0) win[k] = load_vals<V>(x + (k - (W - 1)) * p.ld_x);
        else if (si) win[k] = load_vals<V>(si + k * p.ld_s_in);
    }
    auto load_tile = [&](int t) {
#pragma unroll
        for (int i = 0; i < TT; i++, x += p.ld_x) {
#pragma unroll
            for (int e = 0; e < V; e++) next[i].v[e] = 0.f;
            if (t + i < t1) next[i] = load_vals<V>(x);
        }
    };
    load_tile(t0);
    if (state) {
        const float *xs = p.x + (long long)p.T * d * p.ld_x + s;
#pragma unroll
        for (int k = 0; k < W - 1; k++) {
            Vals<V> ns;
#pragma unroll
            for (int e = 0; e < V; e++) {
                const int t = len[e] - (W - 1) + k;  // its time; before 0 it is win[t + W - 1]
                float v = 0.f;
                if (TT == 1) {
                    v = !len[e] ? win[k].v[e] : k + 1 < W - 1 ? win[k + 1].v[e] : next[0].v[e];
                } else if (t >= 0) {
                    v = xs[t * p.ld_x + e];
                } else {
#pragma unroll
                    for (int q = 0; q < W - 1; q++)
                        if (t + W - 1 == q) v = win[q].v[e];
                }
                ns.v[e] = v;
            }
            store_vals<V>(p.s_out + ((long long)(W - 1) * d + k) * p.ld_s_out + s, ns);
        }
    }
    float *y = p.y + ((long long)p.T * d + t0) * p.ld_y + s;
    for (int t = t0; t < t1; t += TT) {
#pragma unroll
        for (int i = 0; i < TT; i++) win[W - 1 + i] = next[i];
        if (TT > 1 && t + TT < t1) load_tile(t + TT);
#pragma unroll
        for (int i = 0; i < TT; i++, y += p.ld_y) {
            if (t + i >= t1) break;
            Vals<V> o;
#pragma unroll
            for (int e = 0; e < V; e++) {
                float v = b;
#pragma unroll
                for (int k = 0; k < W; k++) v = fmaf(w[k], win[i + k].v[e], v);
                o.v[e] = p.silu ? silu(v) : v;
            }
            if (t + i < least) store_vals<V>(y, o);
            else
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (t + i < len[e]) y[e] = o.v[e];
        }
#pragma unroll
        for (int k = 0; k < W - 1; k++) win[k] = win[TT + k];
    }
}

// Few samples (n < 32): a channel's steps lie next to each other, and a CTA takes
// kFlat runs of 256 / n steps of one channel, lane by lane (sample fastest), so that
// the taps' reads are coalesced at every shift and a thread keeps its sample.  Only
// the first run of a channel (8 steps or more, W <= 8) reads the old state, and its
// CTA writes the new one after that.
constexpr int kFlat = 8;
static_assert(kThreads / 31 >= kMaxConvWidth - 1, "the first run covers the state's reach");

template <int W>
__global__ void __launch_bounds__(kThreads) causal_conv_flat_kernel(const CausalConvArgs p, int blocks) {
    const int d = blockIdx.x / blocks, blk = blockIdx.x - d * blocks, n = (int)p.n;
    const int run = kThreads / n, tl = threadIdx.x / n, s = threadIdx.x - tl * n, t0 = blk * kFlat * run + tl;
    const int len = tl < run ? clamp_len(p.lens, s, p.T) : 0;
    float w[W];
#pragma unroll
    for (int k = 0; k < W; k++) w[k] = __ldg(p.w + d * W + k);
    const float b = p.bias ? __ldg(p.bias + d) : 0.f;
    const float *x = p.x + (long long)p.T * d * p.ld_x + s, *at = x + (t0 - (W - 1)) * p.ld_x;
    const float *si = p.s_in ? p.s_in + (long long)(W - 1) * d * p.ld_s_in + s : nullptr;
    const long long xstep = run * p.ld_x, ystep = run * p.ld_y;
    float v[kFlat][W];
#pragma unroll
    for (int i = 0; i < kFlat; i++, at += xstep) {
        if (t0 + i * run >= len) break;
        if (i == 0 && blk == 0) {
#pragma unroll
            for (int k = 0; k < W; k++) {
                const int t = t0 - (W - 1) + k;
                v[i][k] = t >= 0 ? at[k * p.ld_x] : si ? si[(t + W - 1) * p.ld_s_in] : 0.f;
            }
        } else {
#pragma unroll
            for (int k = 0; k < W; k++) v[i][k] = at[k * p.ld_x];
        }
    }
    if (blk == 0 && W > 1 && p.s_out) {
        // entry k of sample s: the input at len - (W-1) + k, still the old state's before step 0
        const bool on = tl < W - 1;
        const int t = len - (W - 1) + tl;
        const float ns = !on ? 0.f : t >= 0 ? x[t * p.ld_x] : si ? si[(t + W - 1) * p.ld_s_in] : 0.f;
        __syncthreads();
        if (on) p.s_out[((long long)(W - 1) * d + tl) * p.ld_s_out + s] = ns;
    }
    float *y = p.y + ((long long)p.T * d + t0) * p.ld_y + s;
#pragma unroll
    for (int i = 0; i < kFlat; i++, y += ystep) {
        if (t0 + i * run >= len) break;
        float r = b;
#pragma unroll
        for (int k = 0; k < W; k++) r = fmaf(w[k], v[i][k], r);
        *y = p.silu ? silu(r) : r;
    }
}

// ---- selective scan --------------------------------------------------------------
// Both kernels keep the states of a (sample, channel) in one thread's registers, two
// states to a packed register pair, and walk the steps in order; what differs is how
// samples lie across the lanes and how the operands reach them.
//   PASS 0: the whole length in one go.  PASS 1: a chunk from a zero state, leaving
//   its final state and summed step; PASS 2: a chunk from the state it starts in.
typedef unsigned long long f2;  // two fp32 values

__device__ __forceinline__ f2 pack2(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(f2 v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ unsigned smem_addr(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
// asynchronous copies; with `on` false the destination is filled with zeros and
// nothing is read
__device__ __forceinline__ void cp_async16(void *dst, const float *src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_addr(dst)), "l"(src), "r"(on ? 16 : 0));
}
__device__ __forceinline__ void cp_async4(void *dst, const float *src, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(smem_addr(dst)), "l"(src), "r"(on ? 4 : 0));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

// The states of one channel: A log2 e and h, NP of them (the ones beyond N rest at
// zero with A = 0, B = C = 0).
template <int NP>
struct States {
    f2 A[NP / 2], h[NP / 2];
};

template <int NP, int PASS>
__device__ __forceinline__ void load_states(const ScanArgs &p, int d, long long s, int c, bool live, States<NP> &q) {
#pragma unroll
    for (int j = 0; j < NP; j += 2) {
        float a[2], h[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const bool on = live && j + e < p.N;
            a[e] = on ? __ldg(p.A + (long long)d * p.N + j + e) * kLog2e : 0.f;
            h[e] = 0.f;
            if (PASS == 0 && on && p.h0) h[e] = p.h0[((long long)p.N * d + j + e) * p.ld_h0 + s];
            if (PASS == 2 && on) h[e] = p.ws_h[(((long long)c * p.N + j + e) * p.D + d) * p.n + s];
        }
        q.A[j / 2] = pack2(a[0], a[1]);
        q.h[j / 2] = pack2(h[0], h[1]);
    }
}

template <int NP, int PASS>
__device__ __forceinline__ void store_states(const ScanArgs &p, int d, long long s, int c, float sum, const States<NP> &q) {
    if (PASS == 0 && !p.hn) return;
#pragma unroll
    for (int j = 0; j < NP; j += 2) {
        float h[2];
        unpack2(q.h[j / 2], h[0], h[1]);
#pragma unroll
        for (int e = 0; e < 2; e++)
            if (j + e < p.N) {
                if (PASS == 0) p.hn[((long long)p.N * d + j + e) * p.ld_hn + s] = h[e];
                else p.ws_h[(((long long)c * p.N + j + e) * p.D + d) * p.n + s] = h[e];
            }
    }
    if (PASS == 1) p.ws_d[((long long)c * p.D + d) * p.n + s] = sum;
}

// Two states' update; `half`: the second is beyond N (and stays zero also where
// the input is infinite).
template <int PASS>
__device__ __forceinline__ void two_states(f2 A, f2 &h, f2 delta, f2 u, f2 B, f2 C, f2 &acc, const bool half) {
    float e0, e1;
    unpack2(mul2(delta, A), e0, e1);
    h = fma2(pack2(ex2_approx(e0), ex2_approx(e1)), h, mul2(u, B));
    if (half) {
        unpack2(h, e0, e1);
        h = pack2(e0, 0.f);
        unpack2(C, e0, e1);
        C = pack2(e0, 0.f);
    }
    if (PASS != 1) acc = fma2(C, h, acc);
}

__device__ __forceinline__ float finish(f2 acc, float skip, float x, bool gated, float z) {
    float lo, hi;
    unpack2(acc, lo, hi);
    const float v = fmaf(skip, x, lo + hi);
    return gated ? v * silu(z) : v;
}

// Many samples: lane = sample, warp = two channels, which share every B and C they
// read (one where two sets of states would not fit the registers).  Operands arrive
// by cp.async, kWideT steps at a time, two stages.  16384 samples x 50 steps x 64
// channels of 16 states: 365 us, where the exponentials alone take 225 and DRAM 144;
// bound by latency: at the 16 warps a SM that the states' registers leave, a warp waits
// 6.7 cycles an instruction (of 145 a step and channel), 1.9 of them for fixed
// latencies and 0.9 each for shared memory's queue and for its and the exponential
// unit's results; 57 % of the issue slots and 64 % of the exponential unit are busy.
//
// The exponential unit's factors are a tenth of an ulp small on average, which a state
// that hardly decays adds up over its steps: off by 9e-8 after one step, 7e-7 after 80
// or 300 (2-norm, against 64 bits).
constexpr int kWideT = 4, kWideWarps = 8;

__host__ __device__ constexpr int wide_channels(int np) { return np <= 16 ? 2 : 1; }
__host__ __device__ constexpr int wide_stage_floats(int np) { return kWideT * 32 * (2 * np + 3 * wide_channels(np) * kWideWarps); }

// FULL: N == NP.
template <int NP, bool FULL, int PASS>
__global__ void __launch_bounds__(32 * kWideWarps, NP <= 32 ? 2 : 1) scan_wide_kernel(const ScanArgs p, int blocks_per_group, int vec) {
    extern __shared__ __align__(16) float sm[];
    constexpr int kWide = wide_channels(NP), kStep = kWideT * 32, CH = kWideWarps * kWide;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int N = FULL ? NP : p.N, Dg = p.D / p.G, cbs = blocks_per_group * p.G;
    const int cb = blockIdx.x % cbs, g = cb / blocks_per_group, c = blockIdx.y;
    const long long s0 = (long long)(blockIdx.x / cbs) * 32, s = s0 + lane;
    const int db = g * Dg + (cb % blocks_per_group) * CH, dend = (g + 1) * Dg, d0 = db + warp * kWide;
    const int chans = min(CH, dend - db);
    const bool in = s < p.n;
    const int len = in ? clamp_len(p.lens, s, p.T) : 0;
    const int t0 = c * p.chunk, t1 = min(t0 + p.chunk, __reduce_max_sync(0xffffffffu, len));
    constexpr int stage = wide_stage_floats(NP);
    const int left = (int)min(32LL, p.n - s0);

    States<NP> q[kWide];
    float bias[kWide], skip[kWide], sum[kWide];
#pragma unroll
    for (int k = 0; k < kWide; k++) {
        const bool on = d0 + k < dend;
        load_states<NP, PASS>(p, d0 + k, s, c, in && on, q[k]);
        bias[k] = on && p.dt_bias ? p.dt_bias[d0 + k] : 0.f;
        skip[k] = on && p.skip ? p.skip[d0 + k] : 0.f;
        sum[k] = 0.f;
    }

    // kWideT = 4 rows of 32 samples of one feature are one warp's 16-byte copies;
    // a stage holds the features B [NP], C [NP], x, dt, z [CH], feature r copied by
    // warp r % 8.  The pointers are this lane's places in the next stage to copy.
    const int ce = vec ? (lane & 7) * 4 : lane, ct = vec ? lane >> 3 : 0;
    auto first = [&](const float *base, long long row, long long ld) { return base + (row + t0 + ct + (long long)p.T * warp) * ld + s0 + ce; };
    const float *Bs = first(p.B, (long long)p.T * N * g, p.ld_B), *Cs = first(p.C, (long long)p.T * N * g, p.ld_C);
    const float *xs = first(p.x, (long long)p.T * db, p.ld_x), *ds = first(p.dt, (long long)p.T * db, p.ld_dt);
    const float *zs = p.z ? first(p.z, (long long)p.T * db, p.ld_z) : nullptr;
    const bool whole = vec && left == 32 && chans == CH;  // every copy of a stage is of 16 bytes that are there
    auto copy_rows = [&](float *dst, const float *&at, const float *any, long long ld, auto rows, int valid, int t) {
        constexpr int kRows = decltype(rows)::value, kCount = (kRows + kWideWarps - 1) / kWideWarps;
        const long long step = (long long)p.T * ld * kWideWarps;
        const float *src = at;
        at += kWideT * ld;
        float *o = dst + warp * kStep + ct * 32 + ce;
        if (whole && t + kWideT <= t1) {
#pragma unroll
            for (int i = 0; i < kCount; i++, src += step)
                if (kRows % kWideWarps == 0 || warp + i * kWideWarps < kRows)
                    cp_async16(o + i * kWideWarps * kStep, (FULL || warp + i * kWideWarps < valid) ? src : any, FULL || warp + i * kWideWarps < valid);
            return;
        }
        for (int r = warp; r < kRows; r += kWideWarps, src += step, o += kWideWarps * kStep) {
            if (vec) {
                const bool on = t + ct < t1 && r < valid;
                if (ce + 4 <= left || !on) cp_async16(o, on ? src : any, on);
                else
                    for (int w = 0; w < 4; w++) cp_async4(o + w, ce + w < left ? src + w : any, ce + w < left);
            } else {
#pragma unroll
                for (int tt = 0; tt < kWideT; tt++) {
                    const bool on = r < valid && t + tt < t1 && ce < left;
                    cp_async4(o + tt * 32, on ? src + tt * ld : any, on);
                }
            }
        }
    };
    auto issue = [&](int t, float *dst) {
        constexpr std::integral_constant<int, NP> nstates{};
        constexpr std::integral_constant<int, CH> nchans{};
        copy_rows(dst, Bs, p.B, p.ld_B, nstates, N, t);
        if (PASS != 1) copy_rows(dst + NP * kStep, Cs, p.C, p.ld_C, nstates, N, t);
        float *seq = dst + 2 * NP * kStep;
        copy_rows(seq, xs, p.x, p.ld_x, nchans, chans, t);
        copy_rows(seq + CH * kStep, ds, p.dt, p.ld_dt, nchans, chans, t);
        if (PASS != 1 && p.z) copy_rows(seq + 2 * CH * kStep, zs, p.z, p.ld_z, nchans, chans, t);
        cp_async_commit();
    };

    int buf = 0;
    if (t0 < t1) issue(t0, sm);
    for (int t = t0; t < t1; t += kWideT, buf ^= 1) {
        cp_async_wait<0>();
        __syncthreads();  // the stage has landed, and everyone has left the other one
        if (t + kWideT < t1) issue(t + kWideT, sm + (buf ^ 1) * stage);
        if (d0 >= dend) continue;
        const float *bp = sm + buf * stage + lane, *sp = bp + (2 * NP + warp * kWide) * kStep;
        float *y = p.y + ((long long)p.T * d0 + t) * p.ld_y + s;
        const long long ystep = (long long)p.T * p.ld_y;
        const int stop = min(kWideT, min(len, t1) - t);  // this lane's steps of the stage
#pragma unroll 1
        for (int tt = 0; tt < stop; tt++, bp += 32, sp += 32, y += p.ld_y) {
            float x[kWide];
            f2 dd[kWide], uu[kWide], acc[kWide];
#pragma unroll
            for (int k = 0; k < kWide; k++) {  // (a channel beyond the last computes on whatever lies there)
                x[k] = sp[k * kStep];
                float delta = sp[(CH + k) * kStep] + bias[k];
                if (p.softplus) delta = softplus(delta);
                sum[k] += delta;
                dd[k] = pack2(delta, delta);
                uu[k] = pack2(delta * x[k], delta * x[k]);
                acc[k] = 0;
            }
#pragma unroll
            for (int j = 0; j < NP / 2; j++) {
                if (!FULL && 2 * j >= N) break;
                const f2 B = pack2(bp[2 * j * kStep], bp[(2 * j + 1) * kStep]);
                f2 C = 0;
                if (PASS != 1) C = pack2(bp[(NP + 2 * j) * kStep], bp[(NP + 2 * j + 1) * kStep]);
#pragma unroll
                for (int k = 0; k < kWide; k++)
                    two_states<PASS>(q[k].A[j], q[k].h[j], dd[k], uu[k], B, C, acc[k], !FULL && 2 * j + 1 >= N);
            }
            if (PASS != 1) {
#pragma unroll
                for (int k = 0; k < kWide; k++)
                    if (d0 + k < dend) y[k * ystep] = finish(acc[k], skip[k], x[k], p.z != nullptr, p.z ? sp[(2 * CH + k) * kStep] : 0.f);
            }
        }
    }
    if constexpr (PASS != 2) {
#pragma unroll
        for (int k = 0; k < kWide; k++)
            if (in && d0 + k < dend) store_states<NP, PASS>(p, d0 + k, s, c, sum[k], q[k]);
    }
}

// Few samples: the threads of a CTA are the n samples of a run of channels, lane
// by lane (sample fastest).  A feature's steps lie next to each other then, so
// tiles of `steps` x n values of each channel are copied in rows, each thread reads
// its own values from them, and results leave through the place of dt the same way.
// B and C are turned to [step][sample][state] (4 floats of padding keep the
// 16-byte reads of different samples on different banks).  One record of 4096 steps x
// 1024 channels in 74 chunks: 92 us with both passes and the join, the second pass 45
// (exponentials' floor 17), at the 16 warps a SM that its registers and tiles allow.

// Floats between the channels' tiles: n more than a multiple of 32, so that the
// lanes' values lie on 32 banks as the lanes do
__host__ __device__ constexpr int few_row(int steps, int n) { return ((steps - 1) * n + 31) / 32 * 32 + n; }

template <int NP, bool FULL, int PASS>
__global__ void __launch_bounds__(256) scan_few_kernel(const ScanArgs p, int blocks_per_group, int chans, int steps) {
    extern __shared__ __align__(16) float sm[];
    constexpr int kRow = NP + 4;
    const int N = FULL ? NP : p.N, n = (int)p.n, Dg = p.D / p.G, g = blockIdx.x / blocks_per_group, c = blockIdx.y;
    const int db = g * Dg + (blockIdx.x % blocks_per_group) * chans, nch = min(chans, (g + 1) * Dg - db);
    const int dl = threadIdx.x / n, s = threadIdx.x - dl * n, d = db + dl;
    const bool in = dl < nch;
    const int tile = steps * n, row = few_row(steps, n), seq = chans * row;
    float *const bs = sm, *const cs = bs + tile * kRow, *const xs = cs + tile * kRow, *const ds = xs + seq, *const zs = ds + seq;
    const int t0 = c * p.chunk, t1 = min(t0 + p.chunk, p.T);
    const int len = in ? min(clamp_len(p.lens, s, p.T), t1) : 0;

    States<NP> q;
    load_states<NP, PASS>(p, d, s, c, in, q);
    const float bias = in && p.dt_bias ? p.dt_bias[d] : 0.f, skip = in && p.skip ? p.skip[d] : 0.f;
    float sum = 0.f;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    // element e of a feature's tile: step e / n, sample e % n
    auto at = [&](int e, long long ld) { return ld == n ? (long long)e : e / n * ld + e % n; };
    // A tile's features are shared out to the warps, several to one where a tile has
    // fewer than 32 values; long tiles one feature at a time (more than 64 values: 89
    // against 140 us for 37 records of 777 steps).
    auto copy = [&](float *dst, int estride, int rstride, const float *src, long long ld, int rows, int cnt) {
        const long long step = (long long)p.T * ld;
        if (cnt > 64) {
            for (int r = warp; r < rows; r += warps) {
                const float *q = src + r * step;
                float *o = dst + r * rstride;
                if (ld == n)
                    for (int e = lane; e < cnt; e += 32) cp_async4(o + e * estride, q + e, true);
                else
                    for (int e = lane; e < cnt; e += 32) cp_async4(o + e * estride, q + at(e, ld), true);
            }
            return;
        }
        const int per = cnt < 32 ? 32 / cnt : 1, r0 = cnt < 32 ? lane / cnt : 0;
        if (r0 >= per) return;
        const int rs = warps * per, rb = warp * per + r0;
        for (int e = cnt < 32 ? lane - r0 * cnt : lane; e < cnt; e += 32) {
            const float *q = src + rb * step + at(e, ld);
            float *o = dst + rb * rstride + e * estride;
#pragma unroll 4
            for (int r = rb; r < rows; r += rs, q += rs * step, o += rs * rstride) cp_async4(o, q, true);
        }
    };
    for (int t = t0; t < t1; t += steps) {
        const int cnt = min(steps, t1 - t) * n;
        __syncthreads();  // the tile before has been read and written out
        const long long bc = (long long)p.T * N * g + t, sd = (long long)p.T * db + t;
        copy(bs, kRow, 1, p.B + bc * p.ld_B, p.ld_B, N, cnt);
        if (PASS != 1) copy(cs, kRow, 1, p.C + bc * p.ld_C, p.ld_C, N, cnt);
        copy(xs, 1, row, p.x + sd * p.ld_x, p.ld_x, nch, cnt);
        copy(ds, 1, row, p.dt + sd * p.ld_dt, p.ld_dt, nch, cnt);
        if (PASS != 1 && p.z) copy(zs, 1, row, p.z + sd * p.ld_z, p.ld_z, nch, cnt);
        cp_async_commit();
        cp_async_wait<0>();
        __syncthreads();
        const int stop = min(steps, len - t);
        for (int tt = 0; tt < stop; tt++) {
            const int e = tt * n + s, o = dl * row + e;
            const float x = xs[o];
            float delta = ds[o] + bias;
            if (p.softplus) delta = softplus(delta);
            sum += delta;
            const f2 dd = pack2(delta, delta), uu = pack2(delta * x, delta * x);
            f2 acc = 0;
#pragma unroll
            for (int j = 0; j < NP / 4; j++) {
                if (!FULL && 4 * j >= N) break;
                const float4 B = *reinterpret_cast<const float4 *>(bs + e * kRow + 4 * j);
                float4 C = make_float4(0.f, 0.f, 0.f, 0.f);
                if (PASS != 1) C = *reinterpret_cast<const float4 *>(cs + e * kRow + 4 * j);
                two_states<PASS>(q.A[2 * j], q.h[2 * j], dd, uu, pack2(B.x, B.y), pack2(C.x, C.y), acc, !FULL && 4 * j + 1 >= N);
                if (FULL || 4 * j + 2 < N)
                    two_states<PASS>(q.A[2 * j + 1], q.h[2 * j + 1], dd, uu, pack2(B.z, B.w), pack2(C.z, C.w), acc, !FULL && 4 * j + 3 >= N);
            }
            if (PASS != 1) ds[o] = finish(acc, skip, x, p.z != nullptr, p.z ? zs[o] : 0.f);
        }
        if (PASS != 1) {
            __syncthreads();
            const long long step = (long long)p.T * p.ld_y;
            auto wanted = [&](int e) { return !p.lens || t + e / n < clamp_len(p.lens, e % n, p.T); };
            if (cnt <= 32) {
                const int per = 32 / cnt, r0 = lane / cnt, e = lane - r0 * cnt;
                if (r0 < per && wanted(e)) {
                    const int rb = warp * per + r0, rs = warps * per;
                    float *y = p.y + sd * p.ld_y + rb * step + at(e, p.ld_y);
                    for (int r = rb; r < nch; r += rs, y += rs * step) *y = ds[r * row + e];
                }
            } else {
                for (int r = warp; r < nch; r += warps) {
                    float *y = p.y + sd * p.ld_y + r * step;
                    for (int e = lane; e < cnt; e += 32)
                        if (wanted(e)) y[at(e, p.ld_y)] = ds[r * row + e];
                }
            }
        }
    }
    if constexpr (PASS != 2)
        if (in) store_states<NP, PASS>(p, d, s, c, sum, q);
}

// One step of many samples: bound by reading and writing the states, so a thread
// takes V samples (V = 4: 16-byte accesses) of a channel, several states' loads in
// flight at once, and a CTA shares B and C between kStepChans channels.  65536
// samples x 64 channels of 16 states: 108 us, 5.6 TB/s.
constexpr int kStepChans = 16;

template <int NP, bool FULL, int V>
__global__ void __launch_bounds__(256, V == 4 ? 3 : 2) scan_step_kernel(const ScanArgs p, int blocks_per_group) {
    __shared__ __align__(16) float bc[2][NP][32 * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, N = FULL ? NP : p.N;
    const int Dg = p.D / p.G, cbs = blocks_per_group * p.G, cb = blockIdx.x % cbs, g = cb / blocks_per_group;
    const int db = g * Dg + cb % blocks_per_group * kStepChans, dend = min((g + 1) * Dg, db + kStepChans);
    const long long s = (long long)(blockIdx.x / cbs) * (32 * V) + V * lane;  // (V = 4: n is a multiple of 4)
    const bool in = s < p.n;
    for (int r = warp; r < 2 * N; r += 8) {
        const int j = r < N ? r : r - N;
        const float *src = r < N ? p.B + (j + (long long)N * g) * p.ld_B : p.C + (j + (long long)N * g) * p.ld_C;
        if (in) store_vals<V>(&bc[r >= N][j][V * lane], load_vals<V>(src + s));
    }
    __syncthreads();
    if (!in) return;
    bool live[V];
    bool any = false;
#pragma unroll
    for (int i = 0; i < V; i++) {
        live[i] = !p.lens || p.lens[s + i] > 0;
        any |= live[i];
    }
    for (int d = db + warp; d < dend; d += 8) {
        // states in flight at once: 8 of four samples leave registers for a third CTA
        // on the SM (65536 samples, 64 channels of 16 states: 119 us with 16, 108 with 8)
        constexpr int kMost = V == 4 ? 8 : 16, kPart = NP < kMost ? NP : kMost;
        Vals<V> x, dt, z, acc, u;
        float skip = 0.f;
        auto load_part = [&](int j0, Vals<V> (&h)[kPart]) {
#pragma unroll
            for (int j = 0; j < kPart; j++) {
#pragma unroll
                for (int i = 0; i < V; i++) h[j].v[i] = 0.f;
                if (p.h0 && (FULL || j0 + j < N)) h[j] = load_vals<V>(p.h0 + ((long long)N * d + j0 + j) * p.ld_h0 + s);
            }
        };
        Vals<V> h[kPart];
        load_part(0, h);
        if (any) {
            x = load_vals<V>(p.x + d * p.ld_x + s);
            dt = load_vals<V>(p.dt + d * p.ld_dt + s);
            if (p.z) z = load_vals<V>(p.z + d * p.ld_z + s);
            const float bias = p.dt_bias ? __ldg(p.dt_bias + d) : 0.f;
            skip = p.skip ? __ldg(p.skip + d) : 0.f;
#pragma unroll
            for (int i = 0; i < V; i++) {
                dt.v[i] += bias;
                if (p.softplus) dt.v[i] = softplus(dt.v[i]);
                u.v[i] = dt.v[i] * x.v[i];
                acc.v[i] = 0.f;
            }
        }
#pragma unroll
        for (int j0 = 0; j0 < NP; j0 += kPart) {
            if (j0) load_part(j0, h);
#pragma unroll
            for (int j = 0; j < kPart; j++) {
                if (!FULL && j0 + j >= N) break;
                if (any) {
                    const float A = __ldg(p.A + (long long)d * N + j0 + j) * kLog2e;
                    const Vals<V> B = load_vals<V>(&bc[0][j0 + j][V * lane]), C = load_vals<V>(&bc[1][j0 + j][V * lane]);
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float n = fmaf(ex2_approx(dt.v[i] * A), h[j].v[i], u.v[i] * B.v[i]);
                        if (live[i]) h[j].v[i] = n;
                        acc.v[i] = fmaf(C.v[i], n, acc.v[i]);
                    }
                }
                if (p.hn) store_vals<V>(p.hn + ((long long)N * d + j0 + j) * p.ld_hn + s, h[j]);
            }
        }
        if (any) {
            float *y = p.y + d * p.ld_y + s;
            bool all = true;
#pragma unroll
            for (int i = 0; i < V; i++) {
                acc.v[i] = fmaf(skip, x.v[i], acc.v[i]);
                if (p.z) acc.v[i] *= silu(z.v[i]);
                all &= live[i];
            }
            if (all) store_vals<V>(y, acc);
            else
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (live[i]) y[i] = acc.v[i];
        }
    }
}

// One step of few samples: one thread a (sample, channel), every operand's load in
// flight at once; what counts is the latency of one trip to memory.
template <int NP, bool FULL>
__global__ void __launch_bounds__(64) scan_step_few_kernel(const ScanArgs p) {
    const int n = (int)p.n, i = blockIdx.x * 64 + threadIdx.x, d = i / n, s = i - d * n, N = FULL ? NP : p.N;
    if (d >= p.D) return;
    const int g = d / (p.D / p.G);
    const bool live = clamp_len(p.lens, s, 1) > 0;
    float A[NP], B[NP], C[NP], h[NP];
#pragma unroll
    for (int j = 0; j < NP; j++) {
        const bool on = FULL || j < N;
        A[j] = on ? __ldg(p.A + (long long)d * N + j) * kLog2e : 0.f;
        h[j] = on && p.h0 ? p.h0[((long long)N * d + j) * p.ld_h0 + s] : 0.f;
        B[j] = on && live ? p.B[(j + (long long)N * g) * p.ld_B + s] : 0.f;
        C[j] = on && live ? p.C[(j + (long long)N * g) * p.ld_C + s] : 0.f;
    }
    if (live) {
        const float x = p.x[d * p.ld_x + s], z = p.z ? p.z[d * p.ld_z + s] : 0.f;
        float delta = p.dt[d * p.ld_dt + s] + (p.dt_bias ? p.dt_bias[d] : 0.f), acc = 0.f;
        if (p.softplus) delta = softplus(delta);
        const float u = delta * x;
#pragma unroll
        for (int j = 0; j < NP; j++) {
            if (!FULL && j >= N) break;
            h[j] = fmaf(ex2_approx(delta * A[j]), h[j], u * B[j]);
            acc = fmaf(C[j], h[j], acc);
        }
        acc = fmaf(p.skip ? p.skip[d] : 0.f, x, acc);
        p.y[d * p.ld_y + s] = p.z ? acc * silu(z) : acc;
    }
    if (p.hn)
#pragma unroll
        for (int j = 0; j < NP; j++)
            if (FULL || j < N) p.hn[((long long)N * d + j) * p.ld_hn + s] = h[j];
}

// A chunk's steps of one state, one after the other, as the scan's kernels take them.
__device__ __noinline__ float walk_chunk(const ScanArgs &p, long long s, int d, int j, int c, float h) {
    const float A = p.A[(long long)d * p.N + j] * kLog2e, bias = p.dt_bias ? p.dt_bias[d] : 0.f;
    const int t1 = min((c + 1) * p.chunk, clamp_len(p.lens, s, p.T));
    for (int t = c * p.chunk; t < t1; t++) {
        const long long row = t + (long long)p.T * d;
        float delta = p.dt[row * p.ld_dt + s] + bias;
        if (p.softplus) delta = softplus(delta);
        const float B = p.B[(t + (long long)p.T * (j + (long long)p.N * (d / (p.D / p.G)))) * p.ld_B + s];
        h = fmaf(ex2_approx(delta * A), h, delta * p.x[row * p.ld_x + s] * B);
    }
    return h;
}

// Joins the chunks: one thread per (sample, channel, state) walks them in order
// and replaces each chunk's own final state by the state it starts in.
//
// A chunk takes h to e^E h + part, E its steps' sum times A.  A state that decays has
// E <= 0, but nothing keeps A or, without softplus, a step from being of the other
// sign: the factor alone may then be beyond fp32 where the product is not, so it is
// applied as its root, twice; it does not reach a state of 0 (a step whose own factor
// is infinite has made `part` NaN already); and where the sum is not finite all the
// same, two large parts that cancel step by step for instance, the steps decide.
__global__ void __launch_bounds__(kThreads) scan_carry_kernel(const __grid_constant__ ScanArgs p) {
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x, nd = p.n * p.D;
    if (i >= nd * p.N) return;
    const long long sd = i % nd, s = sd % p.n;
    const int j = (int)(i / nd), d = (int)(sd / p.n);
    const float half = p.A[(long long)d * p.N + j] * (0.5f * kLog2e);
    float h = p.h0 ? p.h0[((long long)p.N * d + j) * p.ld_h0 + s] : 0.f;
    // kBatch chunks' values are loaded before they are used: one trip to L2 each
    // would otherwise be the kernel's time
    constexpr int kBatch = 16;
    for (int c0 = 0; c0 < p.chunks; c0 += kBatch) {
        float start[kBatch], root[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            const bool on = c0 + i < p.chunks;
            start[i] = on ? p.ws_h[((long long)(c0 + i) * p.N + j) * nd + sd] : 0.f;
            root[i] = on ? p.ws_d[(c0 + i) * nd + sd] : 0.f;
        }
        float end = h;
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            root[i] = ex2_approx(root[i] * half);
            const float next = fmaf(root[i] * end, root[i], start[i]);  // (beyond the last chunk: end)
            start[i] = end;
            end = next;
        }
        // (what is not finite stays so, and a NaN stays one step by step too)
        if (fabsf(end) <= 3.402823466e38f || h != h) {
#pragma unroll
            for (int i = 0; i < kBatch; i++)
                if (c0 + i < p.chunks) p.ws_h[((long long)(c0 + i) * p.N + j) * nd + sd] = start[i];
            h = end;
            continue;
        }
#pragma unroll 1
        for (int c = c0; c < min(c0 + kBatch, p.chunks); c++) {
            float *const own = p.ws_h + ((long long)c * p.N + j) * nd + sd;
            const float part = *own, f = ex2_approx(p.ws_d[c * nd + sd] * half);
            const float next = h == 0.f ? part : fmaf(f * h, f, part);
            *own = h;
            h = fabsf(next) <= 3.402823466e38f || h != h ? next : walk_chunk(p, s, d, j, c, h);
        }
    }
    if (p.hn) p.hn[((long long)p.N * d + j) * p.ld_hn + s] = h;
}

// Which kernel: with lane = sample a last tile that is mostly empty wastes its
// lanes, and below a warp of samples all of them do.
bool scan_is_few(long long n) { return n < 24 || (n < 64 && n * 4 < (n + 31) / 32 * 32 * 3); }

// scan_few_kernel's channels and steps at a time
void few_shape(long long n, int np, int Dg, int *chans, int *steps) {
    *chans = (int)std::min<long long>(Dg, std::max(1LL, (n <= 8 ? 128 : 256) / n));
    const long long step_bytes = n * (2 * (np + 4) + 3 * *chans) * (long long)sizeof(float);
    *steps = (int)std::max(1LL, std::min(std::max(8LL, 32 / n), 88 * 1024 / step_bytes));
}
size_t few_smem(long long n, int np, int chans, int steps) {
    return sizeof(float) * ((size_t)steps * n * 2 * (np + 4) + (size_t)3 * chans * few_row(steps, (int)n));
}
int states_padded(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : kMaxScanStates; }

bool aligned16(const void *q, long long ld) { return !q || ((ld & 3) == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0); }

template <int NP, bool FULL, int V>
cudaError_t launch_step(const ScanArgs &a, cudaStream_t st) {
    const int bpg = (a.D / a.G + kStepChans - 1) / kStepChans;
    const long long blocks = (a.n + 32 * V - 1) / (32 * V) * bpg * a.G;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    scan_step_kernel<NP, FULL, V><<<(unsigned)blocks, 256, 0, st>>>(a, bpg);
    return cudaGetLastError();
}

template <int NP, bool FULL, int PASS>
cudaError_t launch_pass(const ScanArgs &a, cudaStream_t st) {
    const int Dg = a.D / a.G;
    if constexpr (PASS == 0) {
        if constexpr (NP <= 32)  // (more states' operands do not fit the registers)
            if (a.T == 1 && scan_is_few(a.n)) {
                scan_step_few_kernel<NP, FULL><<<(unsigned)((a.n * a.D + 63) / 64), 64, 0, st>>>(a);
                return cudaGetLastError();
            }
        if (a.T == 1 && !scan_is_few(a.n)) {
            // four samples a thread when there are tiles enough for every SM (and
            // their B and C fit the shared memory)
            if constexpr (NP <= 32)
                if (a.n % 4 == 0 && a.n * a.D >= 148LL * 2 * 128 * kStepChans && aligned16(a.x, a.ld_x) && aligned16(a.dt, a.ld_dt) &&
                    aligned16(a.B, a.ld_B) && aligned16(a.C, a.ld_C) && aligned16(a.z, a.ld_z) && aligned16(a.y, a.ld_y) &&
                    aligned16(a.h0, a.ld_h0) && aligned16(a.hn, a.ld_hn))
                    return launch_step<NP, FULL, 4>(a, st);
            return launch_step<NP, FULL, 1>(a, st);
        }
    }
    if (scan_is_few(a.n)) {
        int chans, steps;
        few_shape(a.n, NP, Dg, &chans, &steps);
        const int bpg = (Dg + chans - 1) / chans, threads = (chans * (int)a.n + 31) / 32 * 32;
        const size_t smem = few_smem(a.n, NP, chans, steps);
        scan_few_kernel<NP, FULL, PASS><<<dim3((unsigned)(bpg * a.G), (unsigned)a.chunks), threads, smem, st>>>(a, bpg, chans, steps);
        return cudaGetLastError();
    }
    constexpr int kWide = wide_channels(NP);
    const int bpg = (Dg + kWideWarps * kWide - 1) / (kWideWarps * kWide);
    const int vec = aligned16(a.x, a.ld_x) && aligned16(a.dt, a.ld_dt) && aligned16(a.B, a.ld_B) && aligned16(a.C, a.ld_C) && aligned16(a.z, a.ld_z);
    const size_t smem = 2 * sizeof(float) * (size_t)wide_stage_floats(NP);
    const long long blocks = (a.n + 31) / 32 * bpg * a.G;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    scan_wide_kernel<NP, FULL, PASS><<<dim3((unsigned)blocks, (unsigned)a.chunks), 32 * kWideWarps, smem, st>>>(a, bpg, vec);
    return cudaGetLastError();
}

template <int NP, bool FULL, int PASS>
cudaError_t configure_pass() {
    cudaError_t e = cudaFuncSetAttribute(scan_few_kernel<NP, FULL, PASS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(scan_wide_kernel<NP, FULL, PASS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 2 * (int)sizeof(float) * wide_stage_floats(NP));
    return e;
}
// Has a kernel loaded: under lazy module loading its first launch would do it, which
// may come while a stream is captured.
template <class K>
cudaError_t load_kernel(K *kernel) {
    cudaFuncAttributes at;
    return cudaFuncGetAttributes(&at, kernel);
}
template <int NP, bool FULL>
cudaError_t configure_n() {
    cudaError_t e = configure_pass<NP, FULL, 0>();
    if (e == cudaSuccess) e = configure_pass<NP, FULL, 1>();
    if (e == cudaSuccess) e = configure_pass<NP, FULL, 2>();
    if (e == cudaSuccess) e = load_kernel(scan_step_kernel<NP, FULL, 1>);
    if constexpr (NP <= 32) {
        if (e == cudaSuccess) e = load_kernel(scan_step_kernel<NP, FULL, 4>);
        if (e == cudaSuccess) e = load_kernel(scan_step_few_kernel<NP, FULL>);
    }
    return e == cudaSuccess ? load_kernel(scan_carry_kernel) : e;
}

template <int NP, bool FULL>
cudaError_t launch_scan_n(const ScanArgs &a, cudaStream_t st, int *launches) {
    *launches = 1;
    if (a.chunks == 1) return launch_pass<NP, FULL, 0>(a, st);
    *launches = 3;
    cudaError_t e = launch_pass<NP, FULL, 1>(a, st);
    if (e != cudaSuccess) return e;
    scan_carry_kernel<<<(unsigned)((a.n * a.D * a.N + kThreads - 1) / kThreads), kThreads, 0, st>>>(a);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    return launch_pass<NP, FULL, 2>(a, st);
}

}  // namespace

// A scan runs one thread a (sample, channel) and is bound by the exponentials, which
// about 16 warps a SM keep busy; splitting it over time computes each twice (the
// chunk's own final state, then its outputs).  So it is split when less than a
// quarter of those warps would run, into chunks of 16 steps or
// more (32 with more states, whose joining costs more).
constexpr long long kScanWarps = 148 * 16;

void scan_split(long long n, int T, int D, int N, int *chunk, int *chunks) {
    *chunk = std::max(T, 1);
    *chunks = 1;
    const int least = N <= 16 ? 16 : 32;
    const long long have = scan_is_few(n) ? (n * D + 31) / 32 : (n + 31) / 32 * ((D + wide_channels(states_padded(N)) - 1) / wide_channels(states_padded(N)));
    if (have < 1 || have * 4 > kScanWarps || T < 2 * least) return;
    const int c = (int)std::min<long long>((kScanWarps + have - 1) / have, T / least);
    if (c < 2) return;
    *chunk = (T + c - 1) / c;
    *chunks = (T + *chunk - 1) / *chunk;
}

size_t scan_workspace_bytes(long long n, int T, int D, int N) {
    int chunk, chunks;
    scan_split(n, T, D, N, &chunk, &chunks);
    return chunks == 1 ? 0 : sizeof(float) * (size_t)n * (size_t)D * (size_t)chunks * (size_t)(N + 1);
}

size_t scan_workspace_limit(long long n, int T, int D, int N) {
    size_t most = 0;  // (no scan of more samples than warps to fill is split)
    for (long long k = 1; k <= std::min(n, kScanWarps * 32); k++) most = std::max(most, scan_workspace_bytes(k, T, D, N));
    return most;
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

namespace {

template <int W, int V, int TT>
cudaError_t launch_conv_tiles(const CausalConvArgs &a, cudaStream_t st) {
    const long long groups = (a.n + V - 1) / V;
    // a thread walks its channel's whole length where that leaves 1024 threads a SM,
    // and fewer tiles of it otherwise
    const int tiles = std::max(1, (a.T + TT - 1) / TT);
    const long long want = std::max(1LL, std::min<long long>(tiles, 148LL * 1024 / std::max(1LL, groups * a.D)));
    const int run = (int)((tiles + want - 1) / want), runs = (tiles + run - 1) / run;
    const long long rows = (long long)runs * a.D;
    unsigned bx = 1;
    while (bx < kThreads && bx < groups) bx *= 2;
    const unsigned by = kThreads / bx;
    const long long sblocks = (groups + bx - 1) / bx, blocks = (rows + by - 1) / by * sblocks;
    if (blocks > 0x7fffffffLL || rows > 0x7fffff00LL) return cudaErrorInvalidConfiguration;
    causal_conv_kernel<W, V, TT><<<(unsigned)blocks, dim3(bx, by), 0, st>>>(a, runs, run, (unsigned)sblocks);
    return cudaGetLastError();
}

constexpr int conv_tile(int W) { return W <= 5 ? 4 : W <= 7 ? 6 : 8; }

template <int W>
cudaError_t load_conv_w() {
    cudaError_t e = load_kernel(causal_conv_flat_kernel<W>);
    if (e == cudaSuccess) e = load_kernel(causal_conv_kernel<W, 1, 1>);
    if (e == cudaSuccess) e = load_kernel(causal_conv_kernel<W, 4, 1>);
    if (e == cudaSuccess) e = load_kernel(causal_conv_kernel<W, 1, 8>);
    return e == cudaSuccess ? load_kernel(causal_conv_kernel<W, 4, conv_tile(W)>) : e;
}

template <int W>
cudaError_t launch_conv_w(const CausalConvArgs &a, cudaStream_t st) {
    if (a.n < 32 && a.T * a.n >= 128) {
        const long long steps = kFlat * (kThreads / a.n), blocks = (a.T + steps - 1) / steps;
        if (blocks * a.D > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
        causal_conv_flat_kernel<W><<<(unsigned)(blocks * a.D), kThreads, 0, st>>>(a, (int)blocks);
        return cudaGetLastError();
    }
    // four samples a thread where that leaves threads enough to fill the GPU
    const bool v4 = a.n % 4 == 0 && a.n / 4 * a.D * std::max(1, a.T / 8) >= 148LL * 1024 && aligned16(a.x, a.ld_x) &&
                    aligned16(a.y, a.ld_y) && aligned16(a.s_in, a.ld_s_in) && aligned16(a.s_out, a.ld_s_out);
    if (a.T == 1) return v4 ? launch_conv_tiles<W, 4, 1>(a, st) : launch_conv_tiles<W, 1, 1>(a, st);
    // short tiles leave registers for more warps (16384 histories of 50 steps, 4 taps:
    // 92 us at 8 steps a tile, 80 at 4); they refill the window, W - 1 steps at least
    constexpr int kTile = conv_tile(W);
    return v4 ? launch_conv_tiles<W, 4, kTile>(a, st) : launch_conv_tiles<W, 1, 8>(a, st);
}

}  // namespace

cudaError_t launch_causal_conv(const CausalConvArgs &a, cudaStream_t st) {
    switch (a.W) {
        case 1: return launch_conv_w<1>(a, st);
        case 2: return launch_conv_w<2>(a, st);
        case 3: return launch_conv_w<3>(a, st);
        case 4: return launch_conv_w<4>(a, st);
        case 5: return launch_conv_w<5>(a, st);
        case 6: return launch_conv_w<6>(a, st);
        case 7: return launch_conv_w<7>(a, st);
        case 8: return launch_conv_w<8>(a, st);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t causal_conv_configure(int W) {
    cudaError_t (*const all[])() = {load_conv_w<1>, load_conv_w<2>, load_conv_w<3>, load_conv_w<4>,
                                    load_conv_w<5>, load_conv_w<6>, load_conv_w<7>, load_conv_w<8>};
    return W >= 1 && W <= kMaxConvWidth ? all[W - 1]() : cudaErrorInvalidValue;
}

cudaError_t launch_scan(const ScanArgs &a, cudaStream_t st, int *launches) {
    const bool full = states_padded(a.N) == a.N;
    switch (states_padded(a.N)) {
        case 4: return full ? launch_scan_n<4, true>(a, st, launches) : launch_scan_n<4, false>(a, st, launches);
        case 8: return full ? launch_scan_n<8, true>(a, st, launches) : launch_scan_n<8, false>(a, st, launches);
        case 16: return full ? launch_scan_n<16, true>(a, st, launches) : launch_scan_n<16, false>(a, st, launches);
        case 32: return full ? launch_scan_n<32, true>(a, st, launches) : launch_scan_n<32, false>(a, st, launches);
        default:
            return full ? launch_scan_n<kMaxScanStates, true>(a, st, launches) : launch_scan_n<kMaxScanStates, false>(a, st, launches);
    }
}

cudaError_t scan_configure(int N) {
    const bool full = states_padded(N) == N;
    switch (states_padded(N)) {
        case 4: return full ? configure_n<4, true>() : configure_n<4, false>();
        case 8: return full ? configure_n<8, true>() : configure_n<8, false>();
        case 16: return full ? configure_n<16, true>() : configure_n<16, false>();
        case 32: return full ? configure_n<32, true>() : configure_n<32, false>();
        default: return full ? configure_n<kMaxScanStates, true>() : configure_n<kMaxScanStates, false>();
    }
}

}  // namespace rosenna

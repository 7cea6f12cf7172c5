// Sequence operators and the 8-bit Gemm: parameter blocks and launchers.
//
// Arrays are rows x n floats as everywhere (kernels.cuh); a sequence of T steps
// and F features has row t + T*f, a state of W rows per feature row k + W*f.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace rosenna {

constexpr int kMaxConvWidth = 8;   // taps of the causal convolution
constexpr int kMaxScanStates = 64; // states per channel of the selective scan

// y[t,d] = act(bias[d] + sum_k w[d][k] x[t - W + 1 + k, d]) over each sample's
// first lens[s] steps; inputs before step 0 come from state_in (row k + (W-1)*d
// holds the input W-1-k steps before step 0), zeros without one.
struct CausalConvArgs {
    const float *w, *bias;  // [D][W]; [D] or null
    const float *x;
    long long ld_x;
    float *y;
    long long ld_y;
    const float *s_in;  // or null
    long long ld_s_in;
    float *s_out;  // or null; may be s_in itself
    long long ld_s_out;
    const int *lens;  // [n] or null (all T)
    long long n;
    int T, D, W, silu;
};

// delta = dt + dt_bias (softplus of it); per state j
//   h_j <- exp(delta A[d][j]) h_j + delta B[t,j] x[t,d]
//   y[t,d] = (sum_j C[t,j] h_j + skip[d] x[t,d]) * silu(z[t,d])
// B and C rows are t + T*(j + N*g), channel d reading group d / (D/G).
struct ScanArgs {
    const float *A, *skip, *dt_bias;  // [D][N]; [D] or null; [D] or null
    const float *x, *dt, *B, *C, *z;  // z or null
    long long ld_x, ld_dt, ld_B, ld_C, ld_z;
    float *y;
    long long ld_y;
    const float *h0;  // or null (zeros); row j + N*d
    long long ld_h0;
    float *hn;  // or null; may be h0 itself
    long long ld_hn;
    const int *lens;
    long long n;
    int T, D, N, G, softplus;
    // split over time (scan_split): chunks of `chunk` steps, per chunk c and
    // state the partial state ws_h[((c*N + j)*D + d)*n + s] and the summed step
    // ws_d[(c*D + d)*n + s]; chunks == 1: not split
    int chunk, chunks;
    float *ws_h, *ws_d;
};

// Chunks that a scan of this size is cut into when it has a workspace, and the
// bytes of that workspace (0: it runs unsplit).
void scan_split(long long n, int T, int D, int N, int *chunk, int *chunks);
size_t scan_workspace_bytes(long long n, int T, int D, int N);
size_t scan_workspace_limit(long long n, int T, int D, int N);  // the most that n samples or fewer need
// Sets a->chunk/chunks and the workspace's parts (null: unsplit); n, T, D, N set.
void scan_bind_workspace(ScanArgs *a, void *workspace);

// Load the kernels of a convolution of W taps / a scan of N states on the current
// device and set their shared memory: before the first launch.
cudaError_t causal_conv_configure(int W);
cudaError_t scan_configure(int N);
cudaError_t launch_causal_conv(const CausalConvArgs &a, cudaStream_t st);
// *launches: kernels launched (1, or 3 when split)
cudaError_t launch_scan(const ScanArgs &a, cudaStream_t st, int *launches);

}  // namespace rosenna

// The 8-bit Gemm: y = act(W x + b) with e4m3 operands and a power-of-two scale
// for each block of 128 (weights: 128 x 128; inputs: 128 of a column).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>
#include <vector>

namespace rosenna {

constexpr int kGemm8Block = 128;
constexpr size_t kGemm8TileBytes = (size_t)kGemm8Block * kGemm8Block;

// Packed weights of one layer: 128 x 128 tiles [Mp/128][Kp/128] of e4m3 bytes
// (zero padded), each the K-major 128-byte-swizzled image that the tensor core
// reads (gemm8_tile_offset), and one scale per tile.
struct Gemm8Weights {
    int M = 0, K = 0, Mp = 0, Kp = 0;
    std::vector<uint8_t> q;
    std::vector<float> scale;
    bool far = false;  // a scale is above 2^7: its product with a column's may be beyond fp32
};
// w[m*K + k]; every value finite.
void gemm8_pack(const float *w, int M, int K, Gemm8Weights *out);

struct Gemm8Args {
    const uint8_t *wq;
    const float *ws;
    const float *bias;  // [Mp] or null
    const float *x;     // row k, column c at x[k*ld_x + c]
    long long ld_x;
    float *y;
    long long ld_y;
    long long n;
    int M, K, Mp, Kp, act, far;
    int *err;       // [64] status words on the device, as the other tensor-core kernels' (tc_common.cuh)
    int *err_host;  // or null: receives err[0] when it is set (host memory the device can write)
    uint8_t *xq;    // workspace: quantised tiles [column tile][Kp/128], for a K too long to keep on chip
    float *xs;      // workspace: their scales [Kp/128][n]
};

size_t gemm8_workspace_bytes(long long n, int M, int K);
size_t gemm8_workspace_limit(long long n, int M, int K);  // the most that n columns or fewer need
cudaError_t gemm8_configure();  // cudaErrorInvalidConfiguration: compiled with other registers than its split assumes
cudaError_t launch_gemm8(Gemm8Args a, void *workspace, int num_sms, cudaStream_t st, int *launches);

}  // namespace rosenna

// The operators' C entries (rosenna_b200/csrc/ops.cu, host code) on a CUDA runtime made
// of counters: what a create and a destroy leave behind, also when a call fails.
#include <cuda_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <map>
#include <new>

#include "../../include/rosenna.h"
#include "../../rosenna_b200/csrc/gemm8.cuh"
#include "../../rosenna_b200/csrc/model_files.hpp"
#include "../../rosenna_b200/csrc/seq_ops.cuh"

static int fail_at = 0, calls = 0;  // the fail_at-th CUDA call fails (0: none)
static int live = 0;                // allocations not freed
static int pending = 0;             // copies from pageable memory that may still be on their way
static int deaths = 0;              // frees of what was not allocated
static std::map<void *, int> blocks;

static cudaError_t step() { return ++calls == fail_at ? cudaErrorUnknown : cudaSuccess; }
static cudaError_t take(void **p, size_t n) {
    cudaError_t e = step();
    if (e != cudaSuccess) return e;
    *p = std::malloc(n);
    blocks[*p]++;
    live++;
    return e;
}
static cudaError_t give(void *p) {
    if (!p) return cudaSuccess;
    if (!blocks.count(p)) deaths++;
    else {
        blocks.erase(p);
        live--;
        std::free(p);
    }
    return cudaSuccess;
}
static cudaError_t wait() {
    cudaError_t e = step();
    if (e == cudaSuccess) pending = 0;
    return e;
}

extern "C" {
cudaError_t cudaGetDeviceCount(int *n) { *n = 1; return step(); }
cudaError_t cudaGetDevice(int *d) { *d = 0; return step(); }
cudaError_t cudaSetDevice(int) { return step(); }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char *cudaGetErrorString(cudaError_t) { return "made up"; }
cudaError_t cudaDeviceGetAttribute(int *v, cudaDeviceAttr a, int) { *v = a == cudaDevAttrComputeCapabilityMajor ? 10 : 148; return step(); }
cudaError_t cudaMalloc(void **p, size_t n) { return take(p, n); }
cudaError_t cudaHostAlloc(void **p, size_t n, unsigned) { return take(p, n); }
cudaError_t cudaFree(void *p) { return give(p); }
cudaError_t cudaFreeHost(void *p) { return give(p); }
// returns once the pageable source has been read, which may be before the copy arrives
cudaError_t cudaMemcpy(void *, const void *, size_t, cudaMemcpyKind k) { pending += k == cudaMemcpyHostToDevice; return step(); }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return wait(); }
cudaError_t cudaDeviceSynchronize() { return wait(); }
}

namespace rosenna {
int report_status(const Status &st) { return st.code; }
static cudaError_t launch(cudaError_t e = cudaSuccess) { return e; }
cudaError_t launch_causal_conv(const CausalConvArgs &, cudaStream_t) { return launch(); }
cudaError_t launch_scan(const ScanArgs &, cudaStream_t, int *) { return launch(); }
cudaError_t launch_gemm8(Gemm8Args, void *, int, cudaStream_t, int *) { return launch(); }
cudaError_t causal_conv_configure(int) { return step(); }
cudaError_t scan_configure(int) { return step(); }
cudaError_t gemm8_configure() { return step(); }
size_t scan_workspace_bytes(long long, int, int, int) { return 0; }
size_t gemm8_workspace_bytes(long long, int, int) { return 0; }
void scan_bind_workspace(ScanArgs *, void *) {}
void gemm8_pack(const float *, int M, int K, Gemm8Weights *out) {
    out->M = M;
    out->K = K;
    out->Mp = out->Kp = 128;
    out->q.assign(128 * 128, 0);
    out->scale.assign(1, 1.f);
}
}  // namespace rosenna

// prints, for each kind and failing call: the status, copies pending, blocks left, wrong
// frees; after the destroy of what was created: blocks left, wrong frees
int main() {
    float w[64] = {0};
    for (int kind = 0; kind < 3; kind++)
        for (fail_at = 0;; fail_at++) {
            rosenna_op *op = nullptr;
            calls = live = pending = deaths = 0;
            const int rc = kind == 0   ? rosenna_causal_conv_create(4, 4, w, w, ROSENNA_ACT_SILU, &op)
                           : kind == 1 ? rosenna_scan_create(4, 4, 1, w, w, w, 1, &op)
                                       : rosenna_gemm8_create(4, 4, w, w, ROSENNA_ACT_NONE, &op);
            const int made = calls;
            const int left = live;
            const int at = fail_at;
            fail_at = 0;
            const int rd = rosenna_op_destroy(op);
            std::printf("%d %d %d %d %d %d %d %d\n", kind, at, rc, pending, left, rd, live, deaths);
            fail_at = at;
            if (at > made) break;
        }
    return 0;
}

// C ABI of the operators a solver drives itself (include/rosenna.h): the causal
// convolution, the selective scan and the 8-bit Gemm.  An operator owns its
// weights on one GPU and nothing that a run writes, so runs need no lock.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>
#include <exception>
#include <memory>
#include <new>
#include <string>
#include <vector>

#include "../../include/rosenna.h"
#include "gemm8.cuh"
#include "model_files.hpp"
#include "ops_checks.hpp"
#include "seq_ops.cuh"

namespace rosenna {
int report_status(const Status &st);  // runtime.cu
}
using namespace rosenna;

struct rosenna_op {
    enum Kind { CONV, SCAN, GEMM8 } kind;
    int device = 0, num_sms = 148;
    void *weights = nullptr;
    // addresses within `weights`
    const float *a = nullptr, *b = nullptr, *c = nullptr;  // conv: w, bias; scan: A, skip, dt_bias; gemm8: scales, bias
    const uint8_t *q = nullptr;
    int rows = 0, cols = 0, groups = 1, flag = 0;  // conv: D, W, -, silu; scan: D, N, G, softplus; gemm8: M, K, -, act
    int rows_p = 0, cols_p = 0, far = 0;           // gemm8: M and K padded; Gemm8Weights::far
    // gemm8: status words of the tensor-core kernel's bounded waits, and a host
    // word it copies the first of them to when it is set
    int *err = nullptr, *err_host = nullptr;
};

namespace {

#define CUDA_TRY(expr)                                                                                \
    do {                                                                                              \
        cudaError_t e_ = (expr);                                                                      \
        if (e_ != cudaSuccess)                                                                        \
            return Status::Err(ROSENNA_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e_)); \
    } while (0)

// No exception leaves a C entry.
template <class F>
int guarded(F f) {
    try {
        try {
            return report_status(f());
        } catch (const std::exception &e) {
            return report_status(Status::Err(ROSENNA_ERR_STATE, e.what()));
        }
    } catch (...) {  // not even the message fitted
        return ROSENNA_ERR_STATE;
    }
}

struct OnDevice {  // the operator's GPU current for the scope
    int before = 0;
    cudaError_t status;
    explicit OnDevice(int id) {
        status = cudaGetDevice(&before);
        if (status == cudaSuccess && before != id) status = cudaSetDevice(id);
        else if (status == cudaSuccess) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

Status use_device(rosenna_op *op) {
    int count = 0;
    if (cudaGetDeviceCount(&count) != cudaSuccess || count <= 0) {
        cudaGetLastError();
        return Status::Err(ROSENNA_ERR_NO_DEVICE, "no CUDA device is visible");
    }
    CUDA_TRY(cudaGetDevice(&op->device));
    int major = 0;
    CUDA_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, op->device));
    if (major < 10) return Status::Err(ROSENNA_ERR_NO_DEVICE, "device is not sm_100 (B200)");
    CUDA_TRY(cudaDeviceGetAttribute(&op->num_sms, cudaDevAttrMultiProcessorCount, op->device));
    return Status::Ok();
}

// Uploads the parts (each from a 256-byte boundary) in one block; `at` receives
// their addresses (null for an empty part).  Waits for the copies: cudaMemcpy from
// pageable memory may return before its data has arrived, and the first run may be
// on a stream that does not wait for the default one.
Status upload(rosenna_op *op, const std::vector<std::pair<const void *, size_t>> &parts, std::vector<const void *> *at) {
    size_t total = 0;
    for (auto &p : parts) total += (p.second + 255) / 256 * 256;
    CUDA_TRY(cudaMalloc(&op->weights, total ? total : 256));
    size_t off = 0;
    at->clear();
    cudaError_t e = cudaSuccess;
    for (auto &p : parts) {
        char *dst = static_cast<char *>(op->weights) + off;
        at->push_back(p.second ? dst : nullptr);
        if (p.second && e == cudaSuccess) e = cudaMemcpy(dst, p.first, p.second, cudaMemcpyHostToDevice);
        off += (p.second + 255) / 256 * 256;
    }
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
    if (e != cudaSuccess) {
        cudaFree(op->weights);
        op->weights = nullptr;
        return Status::Err(ROSENNA_ERR_CUDA, std::string("weights upload: ") + cudaGetErrorString(e));
    }
    return Status::Ok();
}

bool all_finite(const float *p, size_t n) {
    uint32_t most = 0;
    for (size_t i = 0; i < n; i++) {
        uint32_t u;
        std::memcpy(&u, p + i, 4);
        most = std::max(most, u & 0x7fffffffu);
    }
    return most < 0x7f800000u;
}

std::pair<const void *, size_t> floats(const float *p, size_t n) { return {p, p ? n * sizeof(float) : 0}; }

}  // namespace

extern "C" {

int rosenna_causal_conv_create(int channels, int width, const float *w, const float *bias, int act, rosenna_op **out) {
    return guarded([&]() -> Status {
        if (!out || !w) return arg("null pointer");
        *out = nullptr;
        if (channels < 1 || channels > 1 << 20) return shape("channels out of range");
        if (width < 1 || width > kMaxConvWidth) return Status::Err(ROSENNA_ERR_UNSUPPORTED, "a causal convolution has 1 to 8 taps");
        if (act != ROSENNA_ACT_NONE && act != ROSENNA_ACT_SILU)
            return Status::Err(ROSENNA_ERR_UNSUPPORTED, "a causal convolution's activation is none or SiLU");
        auto op = std::make_unique<rosenna_op>();
        op->kind = rosenna_op::CONV;
        op->rows = channels;
        op->cols = width;
        op->flag = act == ROSENNA_ACT_SILU;
        Status st = use_device(op.get());
        std::vector<const void *> at;
        if (st.ok()) st = upload(op.get(), {floats(w, (size_t)channels * width), floats(bias, (size_t)channels)}, &at);
        if (!st.ok()) return st;
        const cudaError_t e = causal_conv_configure(width);
        if (e != cudaSuccess) {
            cudaFree(op->weights);
            return Status::Err(ROSENNA_ERR_CUDA, std::string("convolution set-up: ") + cudaGetErrorString(e));
        }
        op->a = static_cast<const float *>(at[0]);
        op->b = static_cast<const float *>(at[1]);
        *out = op.release();
        return Status::Ok();
    });
}

int rosenna_causal_conv_f32(const rosenna_op *op, const rosenna_causal_conv_args *g, void *stream) {
    return guarded([&]() -> Status {
        if (!g) return arg("null arguments");
        const int64_t n = g->n, T = g->T;
        Status st = check_run(op && op->kind == rosenna_op::CONV, n, T, op ? op->rows : 0);
        if (!st.ok()) return st;
        const int D = op->rows, W = op->cols;
        const Array x{"x", g->x, T * D, or_n(g->ld_x, n)}, y{"y", g->y, T * D, or_n(g->ld_y, n)};
        const Array si{"state_in", g->state_in, (int64_t)(W - 1) * D, or_n(g->ld_state_in, n)};
        const Array so{"state_out", g->state_out, (int64_t)(W - 1) * D, or_n(g->ld_state_out, n)};
        const Array lens{"lens", reinterpret_cast<const float *>(g->lens), 1, n};
        for (auto *a : {&x, &y, &si, &so, &lens})
            if (!(st = check_array(*a, n, a == &x || a == &y)).ok()) return st;
        if (!(st = check_overlaps({x, lens}, {y, so}, si, so, n)).ok()) return st;
        if (n == 0) return Status::Ok();
        OnDevice dev(op->device);
        if (dev.status != cudaSuccess) return Status::Err(ROSENNA_ERR_CUDA, "cudaSetDevice failed");
        CausalConvArgs a{};
        a.w = op->a;
        a.bias = op->b;
        a.x = x.p;
        a.ld_x = x.ld;
        a.y = g->y;
        a.ld_y = y.ld;
        a.s_in = si.p;
        a.ld_s_in = si.ld;
        a.s_out = g->state_out;
        a.ld_s_out = so.ld;
        a.lens = g->lens;
        a.n = n;
        a.T = (int)T;
        a.D = D;
        a.W = W;
        a.silu = op->flag;
        CUDA_TRY(launch_causal_conv(a, static_cast<cudaStream_t>(stream)));
        return Status::Ok();
    });
}

int rosenna_scan_create(int channels, int states, int groups, const float *A, const float *skip, const float *dt_bias,
                        int softplus, rosenna_op **out) {
    return guarded([&]() -> Status {
        if (!out || !A) return arg("null pointer");
        *out = nullptr;
        if (channels < 1 || channels > 1 << 20) return shape("channels out of range");
        if (states < 1 || states > kMaxScanStates) return Status::Err(ROSENNA_ERR_UNSUPPORTED, "a selective scan has 1 to 64 states");
        if (groups < 1 || channels % groups) return shape("groups must divide the channels");
        auto op = std::make_unique<rosenna_op>();
        op->kind = rosenna_op::SCAN;
        op->rows = channels;
        op->cols = states;
        op->groups = groups;
        op->flag = softplus != 0;
        Status st = use_device(op.get());
        std::vector<const void *> at;
        if (st.ok())
            st = upload(op.get(), {floats(A, (size_t)channels * states), floats(skip, (size_t)channels), floats(dt_bias, (size_t)channels)}, &at);
        if (!st.ok()) return st;
        const cudaError_t e = scan_configure(states);
        if (e != cudaSuccess) {
            cudaFree(op->weights);
            return Status::Err(ROSENNA_ERR_CUDA, std::string("scan set-up: ") + cudaGetErrorString(e));
        }
        op->a = static_cast<const float *>(at[0]);
        op->b = static_cast<const float *>(at[1]);
        op->c = static_cast<const float *>(at[2]);
        *out = op.release();
        return Status::Ok();
    });
}

int64_t rosenna_scan_workspace_bytes(const rosenna_op *op, int64_t n, int64_t T) {
    int64_t bytes = 0;
    const int rc = guarded([&]() -> Status {
        const Status st = check_run(op && op->kind == rosenna_op::SCAN, n, T, op ? op->rows : 0);
        if (st.ok()) bytes = (int64_t)scan_workspace_bytes(n, (int)T, op->rows, op->cols);
        return st;
    });
    return rc ? -rc : bytes;
}

int rosenna_scan_f32(const rosenna_op *op, const rosenna_scan_args *g, void *stream) {
    return guarded([&]() -> Status {
        if (!g) return arg("null arguments");
        const int64_t n = g->n, T = g->T;
        Status st = check_run(op && op->kind == rosenna_op::SCAN, n, T, op ? op->rows : 0);
        if (!st.ok()) return st;
        const int D = op->rows, N = op->cols, G = op->groups;
        const Array x{"x", g->x, T * D, or_n(g->ld_x, n)}, dt{"dt", g->dt, T * D, or_n(g->ld_dt, n)};
        const Array B{"B", g->B, T * N * G, or_n(g->ld_B, n)}, C{"C", g->C, T * N * G, or_n(g->ld_C, n)};
        const Array z{"z", g->z, T * D, or_n(g->ld_z, n)}, y{"y", g->y, T * D, or_n(g->ld_y, n)};
        const Array h0{"h0", g->h0, (int64_t)N * D, or_n(g->ld_h0, n)}, hn{"hn", g->hn, (int64_t)N * D, or_n(g->ld_hn, n)};
        const Array lens{"lens", reinterpret_cast<const float *>(g->lens), 1, n};
        for (auto *a : {&x, &dt, &B, &C, &z, &y, &h0, &hn, &lens})
            if (!(st = check_array(*a, n, a != &z && a != &h0 && a != &hn && a != &lens)).ok()) return st;
        if (!(st = check_overlaps({x, dt, B, C, z, lens}, {y, hn}, h0, hn, n)).ok()) return st;
        const int64_t need = (int64_t)scan_workspace_bytes(n, (int)T, D, N);
        if (!(st = check_workspace(g->workspace, g->workspace_bytes, need, false, {x, dt, B, C, z, y, h0, hn, lens}, n)).ok()) return st;
        if (n == 0) return Status::Ok();
        OnDevice dev(op->device);
        if (dev.status != cudaSuccess) return Status::Err(ROSENNA_ERR_CUDA, "cudaSetDevice failed");
        ScanArgs a{};
        a.A = op->a;
        a.skip = op->b;
        a.dt_bias = op->c;
        a.x = x.p;
        a.ld_x = x.ld;
        a.dt = dt.p;
        a.ld_dt = dt.ld;
        a.B = B.p;
        a.ld_B = B.ld;
        a.C = C.p;
        a.ld_C = C.ld;
        a.z = z.p;
        a.ld_z = z.ld;
        a.y = g->y;
        a.ld_y = y.ld;
        a.h0 = h0.p;
        a.ld_h0 = h0.ld;
        a.hn = g->hn;
        a.ld_hn = hn.ld;
        a.lens = g->lens;
        a.n = n;
        a.T = (int)T;
        a.D = D;
        a.N = N;
        a.G = G;
        a.softplus = op->flag;
        scan_bind_workspace(&a, need > 0 ? g->workspace : nullptr);
        int launches = 0;
        CUDA_TRY(launch_scan(a, static_cast<cudaStream_t>(stream), &launches));
        return Status::Ok();
    });
}

int rosenna_gemm8_create(int M, int K, const float *w, const float *bias, int act, rosenna_op **out) {
    return guarded([&]() -> Status {
        if (!out || !w) return arg("null pointer");
        *out = nullptr;
        if (M < 1 || K < 1 || M > 1 << 16 || K > 1 << 16) return shape("an 8-bit Gemm has 1 to 65536 rows and columns");
        if (act < ROSENNA_ACT_NONE || act > ROSENNA_ACT_SILU) return arg("unknown activation");
        if (!all_finite(w, (size_t)M * K) || (bias && !all_finite(bias, (size_t)M))) return arg("weights must be finite");
        Gemm8Weights p;
        gemm8_pack(w, M, K, &p);
        auto op = std::make_unique<rosenna_op>();
        op->kind = rosenna_op::GEMM8;
        op->rows = M;
        op->cols = K;
        op->rows_p = p.Mp;
        op->cols_p = p.Kp;
        op->far = p.far;
        op->flag = act;
        Status st = use_device(op.get());
        std::vector<const void *> at;
        const std::vector<int> zeros(64, 0);
        std::vector<float> padded;  // the kernels read whole tiles
        if (bias) {
            padded.assign((size_t)p.Mp, 0.f);
            std::copy(bias, bias + M, padded.begin());
        }
        if (st.ok())
            st = upload(op.get(), {{p.q.data(), p.q.size()}, floats(p.scale.data(), p.scale.size()),
                                   floats(bias ? padded.data() : nullptr, padded.size()),
                                   {zeros.data(), zeros.size() * sizeof(int)}}, &at);
        if (!st.ok()) return st;
        op->q = static_cast<const uint8_t *>(at[0]);
        op->a = static_cast<const float *>(at[1]);
        op->b = static_cast<const float *>(at[2]);
        op->err = static_cast<int *>(const_cast<void *>(at[3]));
        cudaError_t e = gemm8_configure();
        if (e == cudaSuccess) e = cudaHostAlloc(&op->err_host, sizeof(int), cudaHostAllocDefault);
        if (e != cudaSuccess) {
            cudaFree(op->weights);
            return Status::Err(ROSENNA_ERR_CUDA, std::string("8-bit Gemm set-up: ") + cudaGetErrorString(e));
        }
        *op->err_host = 0;
        *out = op.release();
        return Status::Ok();
    });
}

int64_t rosenna_gemm8_workspace_bytes(const rosenna_op *op, int64_t n) {
    int64_t bytes = 0;
    const int rc = guarded([&]() -> Status {
        const Status st = check_run(op && op->kind == rosenna_op::GEMM8, n, 0, op ? std::max(op->rows, op->cols) : 0);
        if (st.ok()) bytes = (int64_t)gemm8_workspace_bytes(n, op->rows, op->cols);
        return st;
    });
    return rc ? -rc : bytes;
}

int rosenna_gemm8_f32(const rosenna_op *op, const rosenna_gemm8_args *g, void *stream) {
    return guarded([&]() -> Status {
        if (!g) return arg("null arguments");
        const int64_t n = g->n;
        Status st = check_run(op && op->kind == rosenna_op::GEMM8, n, 0, op ? std::max(op->rows, op->cols) : 0);
        if (!st.ok()) return st;
        const int M = op->rows, K = op->cols;
        const Array x{"x", g->x, K, or_n(g->ld_x, n)}, y{"y", g->y, M, or_n(g->ld_y, n)};
        const Array none{"", nullptr, 0, 0};
        for (auto *a : {&x, &y})
            if (!(st = check_array(*a, n, true)).ok()) return st;
        if (!(st = check_overlaps({x}, {y}, none, none, n)).ok()) return st;
        const int64_t need = (int64_t)gemm8_workspace_bytes(n, M, K);
        if (!(st = check_workspace(g->workspace, g->workspace_bytes, need, true, {x, y}, n)).ok()) return st;
        if (*(volatile int *)op->err_host)
            return Status::Err(ROSENNA_ERR_CUDA, "an earlier run timed out waiting on its pipeline (wait " + std::to_string(*op->err_host) +
                                                     "); create the operator again");
        if (n == 0) return Status::Ok();
        OnDevice dev(op->device);
        if (dev.status != cudaSuccess) return Status::Err(ROSENNA_ERR_CUDA, "cudaSetDevice failed");
        Gemm8Args a{};
        a.wq = op->q;
        a.ws = op->a;
        a.bias = op->b;
        a.x = x.p;
        a.ld_x = x.ld;
        a.y = g->y;
        a.ld_y = y.ld;
        a.n = n;
        a.M = M;
        a.K = K;
        a.Mp = op->rows_p;
        a.Kp = op->cols_p;
        a.act = op->flag;
        a.far = op->far;
        a.err = op->err;
        a.err_host = op->err_host;
        int launches = 0;
        CUDA_TRY(launch_gemm8(a, g->workspace, op->num_sms, static_cast<cudaStream_t>(stream), &launches));
        return Status::Ok();
    });
}

int rosenna_op_destroy(rosenna_op *op) {
    return guarded([&]() -> Status {
        std::unique_ptr<rosenna_op> own(op);
        if (!own || !own->weights) return Status::Ok();
        OnDevice dev(own->device);
        if (dev.status != cudaSuccess) return Status::Err(ROSENNA_ERR_CUDA, "cudaSetDevice failed");
        CUDA_TRY(cudaFree(own->weights));  // waits for the runs in flight
        if (own->err_host) CUDA_TRY(cudaFreeHost(own->err_host));
        return Status::Ok();
    });
}

}  // extern "C"

"""What is measured of the sequence operators and the 8-bit Gemm: the cases, their inputs, the plain form of each
operator in elementary torch operations, the framework's calls, and the same results in 64 bits.

Arrays are the framework's: rows x n floats with the sample index fastest, the row of time t and feature f being
t + T*f, so a contiguous tensor of shape (features, T, n).

  conv   y[d,t,s] = silu(b[d] + sum_k w[d,k] x[d,t-W+1+k,s]), earlier times from the state (D, W-1, n)
  scan   delta = softplus(dt + dt_bias); h = exp(delta A) h + delta B x; y = (C . h + skip x) silu(z)
  gemm8  y = act(bias + sum over blocks of 128 of 2^(ew + ex) * (e4m3 weights . e4m3 inputs))
"""
import math

import torch

own = False

E4M3_MAX = 448.0


def listed():
    return [
        # one solver step of a streaming surrogate on a single probe: latency of one call
        {"name": "conv_step_1", "op": "conv", "n": 1, "T": 1, "D": 128, "W": 4, "state": True, "ragged": False},
        # one solver step over a large field of samples, the state carried from step to step
        {"name": "conv_step_field", "op": "conv", "n": 65536, "T": 1, "D": 64, "W": 4, "state": True, "ragged": False},
        # histories of 50 steps (the benchmark LSTM's length) for a batch of samples
        {"name": "conv_history", "op": "conv", "n": 16384, "T": 50, "D": 64, "W": 4, "state": False, "ragged": False},
        # a few long records of unequal length, odd sizes, some of them empty
        {"name": "conv_ragged", "op": "conv", "n": 7, "T": 4099, "D": 257, "W": 3, "state": True, "ragged": True},
        # the same four uses of the scan
        {"name": "scan_step_1", "op": "scan", "n": 1, "T": 1, "D": 128, "N": 16, "G": 1, "state": True, "gate": True, "ragged": False},
        {"name": "scan_step_field", "op": "scan", "n": 65536, "T": 1, "D": 64, "N": 16, "G": 1, "state": True, "gate": True, "ragged": False},
        {"name": "scan_history", "op": "scan", "n": 16384, "T": 50, "D": 64, "N": 16, "G": 1, "state": False, "gate": True, "ragged": False},
        # one long record of a wide layer
        {"name": "scan_long", "op": "scan", "n": 1, "T": 4096, "D": 1024, "N": 16, "G": 1, "state": True, "gate": True, "ragged": False},
        {"name": "scan_ragged", "op": "scan", "n": 37, "T": 777, "D": 100, "N": 7, "G": 2, "state": True, "gate": False, "ragged": True},
        # a projection of a single sample: the weights are most of the bytes
        {"name": "gemm8_1", "op": "gemm8", "n": 1, "K": 1024, "M": 2048, "act": "none", "bias": False},
        # a hidden layer of the benchmark's wide MLP over a quarter of its batch
        {"name": "gemm8_mlp", "op": "gemm8", "n": 1048576, "K": 256, "M": 256, "act": "relu", "bias": True},
        # a projection of a wide layer over many samples, odd sizes
        {"name": "gemm8_wide", "op": "gemm8", "n": 33001, "K": 1000, "M": 2040, "act": "none", "bias": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv", "scan", "gemm8"])
    if op == "gemm8":
        K, M = _log(rng, 16, 2048), _log(rng, 8, 2048)
        n = _log(rng, 1, max(1, min(1 << 20, (1 << 28) // max(K, M))))
        n = max(1, min(n, (1 << 36) // (K * M)))
        return {"op": op, "n": n, "K": K, "M": M, "act": rng.choice(["none", "relu", "tanh", "sigmoid", "silu"]), "bias": rng.random() < 0.7}
    form = rng.choice(["step", "history", "long"])
    N = rng.choice([4, 7, 8, 16, 16, 16, 24, 32]) if op == "scan" else 0
    D = _log(rng, 8, 1024)
    if form == "step":
        T, n = 1, _log(rng, 1, max(1, min(1 << 18, (1 << 22) // D)))
    elif form == "history":
        T = _log(rng, 2, 128)
        n = _log(rng, 16, max(16, min(1 << 16, (1 << 29) // (max(N, 16) * D * T))))
    else:
        n = _log(rng, 1, 16)
        T = _log(rng, 256, max(256, min(8192, (1 << 22) // (n * D))))
    case = {"op": op, "n": n, "T": T, "D": D}
    if op == "conv":
        case["W"] = rng.choice([2, 3, 4, 4, 5, 8])
    else:
        case["N"] = N
        case["G"] = rng.choice([g for g in (1, 1, 2, 4) if D % g == 0])
        case["gate"] = rng.random() < 0.7
    case["state"] = form == "step" or rng.random() < 0.5
    case["ragged"] = form != "step" and rng.random() < 0.4
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    f = dict(device="cuda", generator=g)
    n = case["n"]
    st = dict(case)
    if case["op"] == "gemm8":
        K, M = case["K"], case["M"]
        st["w"] = torch.randn((M, K), **f) / math.sqrt(K)
        st["bias"] = 0.1 * torch.randn((M,), **f) if case["bias"] else None
        x = torch.randn((K, n), **f)
        # a few rows an order of magnitude larger than the rest, as activations have
        x *= torch.where(torch.rand((K, 1), **f) < 0.02, 16.0, 1.0)
        st["x"], st["y"] = x, torch.zeros((M, n), device="cuda")
        # the weights as such a program keeps them: 8-bit values and the exponents of their blocks
        st["wq"], st["we"] = _weight_blocks(st["w"])
        if own:
            from rosenna_b200 import api

            st["call"] = api.Gemm8(st["w"].cpu().numpy(), None if st["bias"] is None else st["bias"].cpu().numpy(),
                                   act=case["act"])
            st["ws"] = torch.zeros(max(16, st["call"].workspace_bytes(n)), dtype=torch.uint8, device="cuda")
        return st
    T, D = case["T"], case["D"]
    st["x"] = torch.randn((D, T, n), **f)
    st["y"] = torch.zeros((D, T, n), device="cuda")
    st["lens"] = None
    if case["ragged"]:
        lens = torch.randint(0, T + 1, (n,), **f)
        lens[0] = T
        if n > 1:
            lens[n // 2] = 0
        st["lens"] = lens.to(torch.int32)
    if case["op"] == "conv":
        W = case["W"]
        st["w"] = torch.randn((D, W), **f) / math.sqrt(W)
        st["bias"] = 0.1 * torch.randn((D,), **f)
        st["s0"] = torch.randn((D, W - 1, n), **f) if case["state"] else None
        st["s1"] = torch.zeros((D, W - 1, n), device="cuda") if case["state"] else None
        if own:
            from rosenna_b200 import api

            st["call"] = api.CausalConv(st["w"].cpu().numpy(), st["bias"].cpu().numpy(), act="silu")
        return st
    N, G = case["N"], case["G"]
    st["A"] = -(torch.arange(1, N + 1, device="cuda") * (0.5 + torch.rand((D, N), **f)))
    st["skip"] = torch.randn((D,), **f)
    # steps between 0.001 and 0.1 before the input's own part
    base = torch.exp(math.log(1e-3) + (math.log(0.1) - math.log(1e-3)) * torch.rand((D,), **f))
    st["dt_bias"] = base + torch.log(-torch.expm1(-base))
    st["dt"] = 0.5 * torch.randn((D, T, n), **f)
    st["B"] = torch.randn((G, N, T, n), **f)
    st["C"] = torch.randn((G, N, T, n), **f)
    st["z"] = torch.randn((D, T, n), **f) if case["gate"] else None
    st["h0"] = 0.5 * torch.randn((D, N, n), **f) if case["state"] else None
    st["h1"] = torch.zeros((D, N, n), device="cuda") if case["state"] else None
    if own:
        from rosenna_b200 import api

        st["call"] = api.SelectiveScan(st["A"].cpu().numpy(), skip=st["skip"].cpu().numpy(),
                                       dt_bias=st["dt_bias"].cpu().numpy(), softplus=True, groups=G)
        st["ws"] = torch.zeros(max(16, st["call"].workspace_bytes(n, T)), dtype=torch.uint8, device="cuda")
    return st


def run(st):
    if own:
        return {"conv": _own_conv, "scan": _own_scan, "gemm8": _own_gemm8}[st["op"]](st)
    return {"conv": _plain_conv, "scan": _plain_scan, "gemm8": _plain_gemm8}[st["op"]](st)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own_conv(st):
    st["call"].run(st["n"], st["T"], _ptr(st["x"]), _ptr(st["y"]), state_in=_ptr(st["s0"]), state_out=_ptr(st["s1"]),
                   lens=_ptr(st["lens"]), stream=torch.cuda.current_stream().cuda_stream)
    return (st["y"], st["s1"])


def _own_scan(st):
    st["call"].run(st["n"], st["T"], _ptr(st["x"]), _ptr(st["dt"]), _ptr(st["B"]), _ptr(st["C"]), _ptr(st["y"]),
                   z=_ptr(st["z"]), h0=_ptr(st["h0"]), hn=_ptr(st["h1"]), lens=_ptr(st["lens"]),
                   workspace=_ptr(st["ws"]), workspace_bytes=st["ws"].numel(),
                   stream=torch.cuda.current_stream().cuda_stream)
    return (st["y"], st["h1"])


def _own_gemm8(st):
    st["call"].run(st["n"], _ptr(st["x"]), _ptr(st["y"]), workspace=_ptr(st["ws"]), workspace_bytes=st["ws"].numel(),
                   stream=torch.cuda.current_stream().cuda_stream)
    return st["y"]


# ---- plain forms -----------------------------------------------------------------------------------------------------
def _inside(st):
    """(T, n) truth values: the time is before the sample's length."""
    return torch.arange(st["T"], device="cuda")[:, None] < st["lens"][None, :]


def _plain_conv(st):
    x, w, W, T, n = st["x"], st["w"], st["W"], st["T"], st["n"]
    D = x.shape[0]
    first = st["s0"] if st["s0"] is not None else x.new_zeros((D, W - 1, n))
    ext = torch.cat([first, x], 1)  # times -(W-1) .. T-1
    # tap k of every output at once: (W, D, T, n)
    taps = torch.stack([ext.narrow(1, k, T) for k in range(W)])
    y = (taps * w.t()[:, :, None, None]).sum(0) + st["bias"][:, None, None]
    y = y / (1.0 + torch.exp(-y))
    if st["lens"] is not None:
        y = torch.where(_inside(st), y, 0.0)
    if st["s0"] is None:
        return (y, None)
    ends = torch.full((n,), T, device="cuda") if st["lens"] is None else st["lens"].long()
    at = ends[None, :] + torch.arange(W - 1, device="cuda")[:, None]  # rows of ext that the new state holds
    return (y, torch.gather(ext, 1, at[None].expand(D, W - 1, n)))


def _plain_scan(st):
    x, T, G = st["x"], st["T"], st["G"]
    D, N = st["A"].shape
    v = st["dt"] + st["dt_bias"][:, None, None]
    delta = torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs()))
    if st["lens"] is not None:
        delta = torch.where(_inside(st), delta, 0.0)  # a step of length 0 leaves the state as it is
    Bd = st["B"].repeat_interleave(D // G, 0)  # (D, N, T, n)
    b = Bd.mul_((delta * x)[:, None])
    a = torch.exp(delta[:, None] * st["A"][:, :, None, None])
    if st["h0"] is not None:
        b[:, :, 0] += a[:, :, 0] * st["h0"]
    # the recurrence h = a h + b for all times, by doubling the reach of each time's partial sum
    reach = 1
    while reach < T:
        b = torch.cat([b[:, :, :reach], torch.addcmul(b[:, :, reach:], a[:, :, reach:], b[:, :, :-reach])], 2)
        if 2 * reach < T:
            a = torch.cat([a[:, :, :reach], a[:, :, reach:] * a[:, :, :-reach]], 2)
        reach *= 2
    hn = None if st["h0"] is None else b[:, :, -1].clone()
    del a
    y = (b.view(G, D // G, N, T, -1) * st["C"][:, None]).sum(2).view(D, T, -1) + st["skip"][:, None, None] * x
    if st["z"] is not None:
        y = y * (st["z"] / (1.0 + torch.exp(-st["z"])))
    if st["lens"] is not None:
        y = torch.where(_inside(st), y, 0.0)
    return (y, hn)


def _exponents(amax):
    """The least e >= -126 with amax <= 448 * 2^e (0 where the block is all zeros)."""
    m, q = torch.frexp(amax)  # amax = m 2^q, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.clamp(q - 9 + (m > 0.875).to(q.dtype), min=-126)
    return torch.where(amax > 0, e, 0)


def _two_to(e):
    """2^e as 32-bit floats, exactly, for -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _weight_blocks(w):
    M, K = w.shape
    Mp, Kp = -(-M // 128) * 128, -(-K // 128) * 128
    p = torch.zeros((Mp, Kp), device=w.device)
    p[:M, :K] = w
    e = _exponents(p.view(Mp // 128, 128, Kp // 128, 128).abs().amax((1, 3)))
    q = (p.view(Mp // 128, 128, Kp // 128, 128) * _two_to(-e)[:, None, :, None]).view(Mp, Kp)
    return q.to(torch.float8_e4m3fn), e


def _plain_gemm8(st):
    x, K, M, n = st["x"], st["K"], st["M"], st["n"]
    Mp, Kp = st["wq"].shape
    w = st["wq"].float().view(Mp // 128, 128, Kp // 128, 128) * _two_to(st["we"])[:, None, :, None]
    p = torch.zeros((Kp, n), device="cuda")
    p[:K] = x
    p = p.view(Kp // 128, 128, n)
    amax = p.abs().amax(1, keepdim=True)
    e = _exponents(amax)
    p = (p * _two_to(-e)).to(torch.float8_e4m3fn).float() * torch.where(torch.isfinite(amax), _two_to(e), float("nan"))
    y = torch.matmul(w.view(Mp, Kp)[:M], p.view(Kp, n))
    if st["bias"] is not None:
        y = y + st["bias"][:, None]
    if st["act"] == "relu":
        y = torch.clamp(y, min=0.0)
    elif st["act"] == "tanh":
        y = 1.0 - 2.0 / (1.0 + torch.exp(2.0 * y))
    elif st["act"] == "sigmoid":
        y = 1.0 / (1.0 + torch.exp(-y))
    elif st["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    return y


# ---- what one pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    n = case["n"]
    if case["op"] == "gemm8":
        K, M = case["K"], case["M"]
        return {"bytes": 4 * n * (K + M) + K * M + (4 * M if case["bias"] else 0), "flops": 2 * K * M * n}
    T, D = case["T"], case["D"]
    items = n * T * D
    if case["op"] == "conv":
        W = case["W"]
        state = 8 * n * D * (W - 1) if case["state"] else 0
        return {"bytes": 8 * items + state + 4 * D * (W + 1) + (4 * n if case["ragged"] else 0), "flops": items * (2 * W + 4)}
    N, G = case["N"], case["G"]
    seq = 4 * items * (4 if case["gate"] else 3) + 8 * n * T * N * G
    state = 8 * n * D * N if case["state"] else 0
    return {"bytes": seq + state + 4 * D * (N + 2) + (4 * n if case["ragged"] else 0), "flops": items * (7 * N + 16)}


# ---- 64 bits, step by step as the definitions read -------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "gemm8": _exact_gemm8}[case["op"]](st)


def _exact_conv(st):
    W, T, n = st["W"], st["T"], st["n"]
    x, w, b = st["x"].double(), st["w"].double(), st["bias"].double()
    D = x.shape[0]
    y = b[:, None, None].expand(D, T, n).clone()
    for k in range(W):
        back = W - 1 - k  # this tap reads the input `back` steps earlier
        if back < T:
            y[:, back:] += w[:, k, None, None] * x[:, :T - back]
        if back and st["s0"] is not None:
            m = min(back, T)
            y[:, :m] += w[:, k, None, None] * st["s0"].double()[:, k:k + m]
    y = y * torch.sigmoid(y)
    s1 = None
    if st["s0"] is not None:
        lens = torch.full((n,), T, device="cuda") if st["lens"] is None else st["lens"].long()
        s1 = st["s0"].double().clone()
        for k in range(W - 1):
            t = lens - (W - 1) + k  # time of the state's row k; before 0 it is row t + W-1 of the old state
            old = st["s0"].double().gather(1, (t.clamp(max=-1) + W - 1).clamp(min=0)[None, None].expand(D, 1, n))[:, 0]
            new = x.gather(1, t.clamp(min=0, max=T - 1)[None, None].expand(D, 1, n))[:, 0]
            s1[:, k] = torch.where(t >= 0, new, old)
    if st["lens"] is not None:
        y[(torch.arange(T, device="cuda")[:, None] >= st["lens"][None])[None].expand(D, T, n)] = 0.0
    return (y, s1)


def _exact_scan(st):
    T, n, G = st["T"], st["n"], st["G"]
    A = st["A"].double()
    D, N = A.shape
    group = torch.arange(D, device="cuda") // (D // G)
    h = torch.zeros((D, N, n), dtype=torch.float64, device="cuda") if st["h0"] is None else st["h0"].double()
    y = torch.zeros((D, T, n), dtype=torch.float64, device="cuda")
    for t in range(T):
        delta = torch.nn.functional.softplus(st["dt"][:, t].double() + st["dt_bias"].double()[:, None], threshold=50.0)
        x = st["x"][:, t].double()
        new = torch.exp(delta[:, None] * A[:, :, None]) * h + (delta * x)[:, None] * st["B"][:, :, t].double()[group]
        out = torch.einsum("djn,djn->dn", new, st["C"][:, :, t].double()[group]) + st["skip"].double()[:, None] * x
        if st["z"] is not None:
            out = out * torch.nn.functional.silu(st["z"][:, t].double())
        if st["lens"] is None:
            h, y[:, t] = new, out
        else:
            live = t < st["lens"]
            h = torch.where(live, new, h)
            y[:, t] = torch.where(live, out, 0.0)
    return (y, None if st["h0"] is None else h)


def _double_power(k):
    """2^k for whole k, in 64 bits, exactly."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _e4m3(v):
    """v (64 bits) rounded to the nearest e4m3 value, ties to even."""
    step = _double_power(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0) - 3.0)
    return torch.clamp(torch.round(v / step) * step, -E4M3_MAX, E4M3_MAX)


def _power(amax):
    """The power of two that a block with this largest magnitude is divided by."""
    p = _double_power(torch.ceil(torch.log2(amax.clamp(min=1e-45) / E4M3_MAX)))
    p = torch.where(amax > p * E4M3_MAX, 2 * p, torch.where(amax <= p / 2 * E4M3_MAX, p / 2, p))  # the logarithm's rounding
    return torch.where(amax > 0, p.clamp(min=2.0 ** -126), 1.0)


def _exact_gemm8(st):
    K, M, n = st["K"], st["M"], st["n"]
    x, w = st["x"].double(), st["w"].double()
    y = torch.zeros((M, n), dtype=torch.float64, device="cuda")
    for k in range(0, K, 128):
        xb = x[k:k + 128]
        px = _power(xb.abs().amax(0, keepdim=True))
        xq = _e4m3(xb / px) * px
        wq = torch.empty_like(w[:, k:k + 128])
        for m in range(0, M, 128):
            wb = w[m:m + 128, k:k + 128]
            pw = _power(wb.abs().amax())
            wq[m:m + 128] = _e4m3(wb / pw) * pw
        y += wq @ xq
    if st["bias"] is not None:
        y += st["bias"].double()[:, None]
    f = {"none": lambda v: v, "relu": torch.relu, "tanh": torch.tanh, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}
    return f[st["act"]](y)

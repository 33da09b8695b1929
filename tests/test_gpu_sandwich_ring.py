"""The sandwich norms' kernels for many rows of whole vectors (loads by bulk copies) in the layouts and types
that a caller may give them: rows of any pitch, broadcast rows and gates, weights in fp32, rows that hold
no numbers, a stream written over an input, and a captured step.  Tolerances: test_gpu_sandwich_norm."""
import ctypes

import pytest
import torch

import kernel_opt
from _helpers import CAPI_LIB
from test_gpu_sandwich_norm import DTYPES, E, EPS, GATES, check_forward, check_grads, inputs, run, within

pytestmark = pytest.mark.gpu


def check_eight_bits(t, stream):
    q, scales, s8 = kernel_opt.fused_sandwich_rmsnorm_fp8(**{k: None if v is None else v.detach() for k, v in t.items()},
                                                          eps=EPS)
    assert torch.equal(s8, stream)
    h = stream.shape[-1]
    s = stream.double()
    v = s / (s.square().mean(-1, keepdim=True) + EPS).sqrt() * t["weight"].double()
    step = scales.double().repeat_interleave(128, -1)[..., :h]
    top = torch.nn.functional.pad(v.abs(), (0, -h % 128)).unflatten(-1, (-1, 128)).amax(-1) / 448
    within(scales, top, 44 * E * top, "scales")
    within(q.double() * step, v, torch.maximum(v.abs() / 16, step / 1024) * (1 + 100 * E) + 100 * E * v.abs(), "q")


def views(dtype, n, h, gate):
    """Inputs of one shape in several layouts: whole vectors, at other pitches and starts."""
    u = 16 // dtype.itemsize
    t, gy, gs = inputs(n, h, dtype, gate)

    def pitched(a, before, after):
        wide = torch.zeros(a.shape[0], before + a.shape[1] + after, device="cuda", dtype=a.dtype)
        wide[:, before:before + a.shape[1]] = a
        return wide[:, before:before + a.shape[1]]

    yield t, gy, gs
    yield ({**t, "x": pitched(t["x"], u, 2 * u), "residual": pitched(t["residual"], 3 * u, 0),
            "gate": pitched(t["gate"], 0, 5 * u) if gate in ("full", "token") else t["gate"]},
           pitched(gy, 2 * u, u), pitched(gs, 0, u))
    yield ({**t, "x": t["x"][:1].expand(n, h), "gate": t["gate"][:1].expand(n, h) if gate == "full" else t["gate"]},
           gy[:1].expand(n, h), gs)
    yield {**t, "residual": t["residual"][:1].expand(n, h)}, gy, gs[:1].expand(n, h)
    if gate == "token":
        yield {**t, "gate": t["gate"][:1].expand(n, 1)}, gy, gs


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("n,h", [(700, 256), (460, 2048), (301, 3584), (299, 8192)])
def test_layouts(dtype, gate, n, h):
    for t, gy, gs in views(dtype, n, h, gate):
        y, stream, got = run(t, gy, gs, 1.0, 1.0)
        check_forward(t, y, stream, 1.0, 1.0)
        check_grads(t, stream, gy, gs, got, 1.0, 1.0)
        check_eight_bits(t, stream)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("n,h", [(700, 1000), (300, 3584), (299, 8192)])
def test_weights_in_fp32(dtype, gate, n, h):
    t, gy, gs = inputs(n, h, dtype, gate, torch.float32)
    y, stream, got = run(t, gy, gs, 1.0, 1.0)
    check_forward(t, y, stream, 1.0, 1.0)
    check_grads(t, stream, gy, gs, got, 1.0, 1.0)
    check_eight_bits(t, stream)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("h", [520, 3584])
def test_zeros_infinities_and_nan_stay_in_their_rows(dtype, h):
    # every seventh row of four kinds, so that a group's rows before and after one are sound
    n = 2003
    t, gy, gs = inputs(n, h, dtype, "token")
    t["x"][0::28] = 0
    t["x"][7::28, 7] = torch.nan
    t["residual"][14::28, 9] = torch.inf
    t["gate"][21::28] = 0
    y, stream, got = run(t, gy, gs, 1.0, 1.0, ("x", "residual", "gate"))
    sound = torch.ones(n, dtype=torch.bool, device="cuda")
    sound[7::28] = sound[14::28] = False
    part = {k: (v[sound] if k in ("x", "residual", "gate") else v) for k, v in t.items()}
    check_forward(part, y[sound], stream[sound], 1.0, 1.0)
    check_grads(part, stream[sound], gy[sound], gs[sound], {k: v[sound] for k, v in got.items()}, 1.0, 1.0)
    assert stream[7::28].isnan().all() and y[14::28].isnan().any(1).all()
    q, scales, s8 = kernel_opt.fused_sandwich_rmsnorm_fp8(**{k: v.detach() for k, v in t.items()}, eps=EPS)
    assert torch.equal(s8[sound], stream[sound]) and scales[sound].isfinite().all() and q.float()[sound].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n,h", [(40, 1024), (17, 2051), (700, 3584), (299, 8192), (200, 16384)])
def test_stream_over_an_input(dtype, eight, n, h):
    # the C ABI allows the stream to be x or the residual
    i64, p, c_int, c_float = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    lib = ctypes.CDLL(CAPI_LIB)
    lib.k1_last_error.restype = ctypes.c_char_p
    f = lib.k1_sandwich_rmsnorm_fp8 if eight else lib.k1_sandwich_rmsnorm
    f.argtypes = [p, i64, p, i64, p, p, c_int, i64, p, c_int, c_int, i64, i64, c_float, c_float, c_float, p, p, p, p] + \
        ([] if eight else [p])
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    t, _, _ = inputs(n, h, dtype, "none")
    results = []
    for over in ("own", "x", "residual"):
        a, b = t["x"].clone(), t["residual"].clone()
        stream = {"own": torch.empty_like(a), "x": a, "residual": b}[over]
        out = torch.empty(n, h, dtype=torch.uint8 if eight else dtype, device="cuda")
        scales = torch.empty(n, -(-h // 128), device="cuda")
        tail = [scales.data_ptr()] if eight else [None, None]
        rc = f(a.data_ptr(), h, b.data_ptr(), h, t["post_weight"].data_ptr(), None, 0, 0, t["weight"].data_ptr(), code, code,
               n, h, 1.0, 1.0, EPS, stream.data_ptr(), out.data_ptr(), *tail, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.k1_last_error()
        assert over == "x" or torch.equal(a, t["x"])
        assert over == "residual" or torch.equal(b, t["residual"])
        results.append((stream.clone(), out.clone(), scales.clone() if eight else out))
    for other in results[1:]:
        assert all(torch.equal(u, v) for u, v in zip(results[0], other))


def test_captured():
    n, h = 600, 1024
    t, gy, gs = inputs(n, h, torch.bfloat16, "column")
    t = {k: v.requires_grad_(True) for k, v in t.items()}

    def step():
        out = kernel_opt.fused_sandwich_rmsnorm(**t, branch_scale=0.5)
        return (*out, *torch.autograd.grad(out, list(t.values()), (gy, gs)), *kernel_opt.fused_sandwich_rmsnorm_fp8(**t))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2):
        with torch.no_grad():
            for k, v in inputs(n, h, torch.bfloat16, "column", seed=seed)[0].items():
                t[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))

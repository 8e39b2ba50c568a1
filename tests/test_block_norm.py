"""The norms around a block (block_norm, block_norm_bwd) against 64-bit formulas, 64-bit autograd and differences.

Tolerances.  One rounding to the storage type costs eps/2 of the value (2^-8 bf16, 2^-11 fp16, 2^-24 fp32).  The fp32
arithmetic behind it: a mean of up to 4096 squares, added in chains of at most 4096/32 + 8 terms and a root, relative error
below 140 * 2^-24 = 8.3e-6 in the worst case, about a tenth of that as it happens (errors of random sign); a handful of products more.
1e-5 of the tensor's largest value covers it, the framework's figure for fp32 operators.  A parameter gradient is a sum over
tokens whose chains have at most 64 terms here: 64 * 2^-24 < 4e-6 of the sum of magnitudes, plus the 1e-5 of its factors.
"""
import math

import pytest
import torch

from ane_b200 import dev_ops, lib

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


# ------------------------------------------------------------------ references
def chan(t):
    return 1.0 if t is None else t.double()[..., None] if t.dim() == 2 else t.double()[None, :, None]


def forward64(x, f, w_post, gate, alpha, eps=EPS):
    """x2 before it is rounded."""
    n = f.double()
    if w_post is not None:
        n = n / torch.sqrt((n * n).mean(1, keepdim=True) + eps) * chan(w_post)
    return x.double() + alpha * chan(gate) * n


def norm64(x2, w_pre, eps=EPS):
    z = x2.double()
    return z / torch.sqrt((z * z).mean(1, keepdim=True) + eps) * chan(w_pre)


def grads64(dy, dx2, x2, f, w_pre, w_post, gate, alpha, eps=EPS):
    """By autograd on the 64-bit forward pass: dx, df, dw_pre, dw_post, dgate; the graph starts from x = x2 - branch, so that
    the sum is x2 itself."""
    f, w_pre = f.double().requires_grad_(), w_pre.double().requires_grad_()
    w_post = None if w_post is None else w_post.double().requires_grad_()
    gate = None if gate is None else gate.double().requires_grad_()
    branch = forward64(torch.zeros_like(f), f, w_post, gate, alpha, eps)
    x = (x2.double() - branch.detach()).requires_grad_()
    out = x + branch
    loss = (norm64(out, w_pre, eps) * dy.double()).sum()
    if dx2 is not None:
        loss = loss + (out * dx2.double()).sum()
    leaves = [t for t in (x, f, w_pre, w_post, gate) if t is not None]
    got = dict(zip(map(id, leaves), torch.autograd.grad(loss, leaves)))
    return [None if t is None else got[id(t)] for t in (x, f, w_pre, w_post, gate)]


def within(got, ref, dt, scale=None):
    ref = ref.double()
    tol = torch.finfo(dt).eps / 2 * ref.abs() + 1e-5 * (ref.abs().max() if scale is None else scale) + (2.0 ** -25 if dt == torch.float16 else 0.0)
    worst = ((got.double() - ref).abs() / tol).max()
    return bool(worst <= 1.0), float(worst)


# ------------------------------------------------------------------ CPU
def test_refusals_without_a_gpu():
    x, w = torch.zeros(2, 8, 4), torch.ones(8)
    with pytest.raises(ValueError, match="f: expected"):
        dev_ops.block_norm(x, torch.zeros(2, 8, 5), w)
    with pytest.raises(ValueError, match="w_pre"):
        dev_ops.block_norm(x, x.clone(), torch.ones(7))
    with pytest.raises(ValueError, match="w_post"):
        dev_ops.block_norm(x, x.clone(), w, w_post=torch.ones(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="gate"):
        dev_ops.block_norm(x, x.clone(), w, gate=torch.ones(3, 8))
    with pytest.raises(ValueError, match="current CUDA device"):
        dev_ops.block_norm(x, x.clone(), w)
    with pytest.raises(ValueError, match="dgate needs gate"):
        dev_ops.block_norm_bwd(x, x.clone(), x.clone(), w, None, dgate=torch.ones(8))
    with pytest.raises(ValueError, match="dx2"):
        dev_ops.block_norm_bwd(x, x.clone(), x.clone(), w, None, dx2=x.bfloat16())


def test_the_library_refuses_before_init():
    if torch.cuda.is_available():
        return
    L = lib.load()
    assert L.ane_cuda_block_norm_dev(None, 0, 1, 1, 1, None, None, None, None, None, None, 0, None, 1.0, 1e-5) == lib.ERR_NOT_INIT
    assert L.ane_cuda_block_norm_bwd_dev(None, 0, 1, 1, 1, *[None] * 11, 0, None, 1.0, 1e-5) == lib.ERR_NOT_INIT


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    lib.init(0)
    return dev_ops


def inputs(shape, dt, post, gate, seed=0):
    B, C, S = shape
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def r(*s, scale=1.0, shift=0.0, dtype=torch.float32):
        return (torch.randn(s, generator=g, device="cuda") * scale + shift).to(dtype)
    s = dict(x=r(B, C, S, dtype=dt), f=r(B, C, S, scale=2.0, dtype=dt), w_pre=r(C, scale=0.1, shift=1.0), w_post=r(C, scale=0.1, shift=1.0) if post else None,
             gate=None if gate == "none" else r(*((B, C) if gate == "sequence" else (C,)), scale=0.4, shift=0.3))
    return s, r


SHAPES = [(1, 1, 1), (2, 7, 3), (3, 33, 5), (1, 768, 256), (2, 128, 257), (3, 100, 333), (4, 64, 1), (1, 4096, 64), (2, 1024, 48), (70, 16, 2),
          (1, 300, 8), (1, 129, 64), (1, 4099, 8), (3, 2048, 72), (2, 1024, 1032), (1, 6000, 16),
          (3, 1147, 38), (2, 1025, 333), (1, 2047, 17), (1, 2049, 17), (40, 50, 1001),
          (32, 1024, 512), (40, 96, 1000), (20, 1000, 264), (24, 700, 520)]      # many tiles: the pipelined forms


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "sequence"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(ops, shape, dt, post, gate):
    s, _ = inputs(shape, DT[dt], post, gate)
    x2, y = ops.block_norm(s["x"], s["f"], s["w_pre"], w_post=s["w_post"], gate=s["gate"], alpha=0.35, eps=EPS)
    assert within(x2, forward64(s["x"], s["f"], s["w_post"], s["gate"], 0.35), DT[dt])[0]
    assert within(y, norm64(x2, s["w_pre"]), DT[dt])[0]
    # in place, the same bits
    x = s["x"].clone()
    a, b = ops.block_norm(x, s["f"], s["w_pre"], w_post=s["w_post"], gate=s["gate"], alpha=0.35, eps=EPS, x2=x)
    assert torch.equal(a, x2) and torch.equal(b, y)
    assert lib.poll_status().wait_giveups == 0


@pytest.mark.gpu
@pytest.mark.parametrize("with_dx2", [True, False])
@pytest.mark.parametrize("gate", ["none", "channel", "sequence"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(ops, shape, dt, post, gate, with_dx2):
    dt = DT[dt]
    s, r = inputs(shape, dt, post, gate, seed=1)
    B, C, S = shape
    dy, dx2 = r(B, C, S, dtype=dt), r(B, C, S, dtype=dt) if with_dx2 else None
    acc = [r(C), r(C) if post else None, None if s["gate"] is None else r(*s["gate"].shape)]
    got = [None if t is None else t.clone() for t in acc]
    args = (dy, s["x"], s["f"], s["w_pre"])
    kw = dict(w_post=s["w_post"], gate=s["gate"], dx2=dx2, alpha=0.35, eps=EPS)
    dx, df = ops.block_norm_bwd(*args, got[0], dw_post=got[1], dgate=got[2], **kw)
    ref = grads64(dy, dx2, s["x"], s["f"], s["w_pre"], s["w_post"], s["gate"], 0.35)
    # the parts of dx: what cancels in it does not shrink its error
    z = s["x"].double()
    r2 = 1 / torch.sqrt((z * z).mean(1, keepdim=True) + EPS)
    size = max(float((dy.double() * chan(s["w_pre"]) * r2).abs().max()), float(ref[0].abs().max()))
    rf = 1 / torch.sqrt((s["f"].double() ** 2).mean(1, keepdim=True) + EPS) if post else torch.ones_like(r2)
    scale_f = 0.35 * size * float((chan(s["gate"]) * rf * torch.ones_like(rf)).abs().max()) * 1.5
    assert within(dx, ref[0], dt, size)[0], within(dx, ref[0], dt, size)
    assert within(df, ref[1], dt, max(scale_f, float(ref[1].abs().max())))[0]
    terms = [(dy.double() * z * r2).abs().sum((0, 2)), None, None]
    # dx enters these two sums with the error of its parts, 1e-5 of their size, however much of them cancels
    parts = ref[0].abs() + size
    if post:
        terms[1] = (0.35 * parts * s["f"].double() * rf * chan(s["gate"])).abs().sum((0, 2))
    if s["gate"] is not None:
        d = (0.35 * parts * (s["f"].double() * rf * chan(s["w_post"])).abs()).sum(2)
        terms[2] = d if gate == "sequence" else d.sum(0)
    for name, a, b, t, before in zip(("dw_pre", "dw_post", "dgate"), got, ref[2:], terms, acc):
        if a is not None:
            err = (a.double() - before.double() - b).abs()
            bound = 1.4e-5 * (t + t.max()) + 2.0 ** -23 * (before.double().abs() + b.abs())
            assert bool((err <= bound).all()), (name, float((err / bound).max()))
    # without the parameter gradients, over dx2 and f: the same bits; again: the same bits
    again = [None if t is None else t.clone() for t in acc]
    dx_, df_ = ops.block_norm_bwd(*args, again[0], dw_post=again[1], dgate=again[2], **kw)
    assert torch.equal(dx, dx_) and torch.equal(df, df_) and all(a is None or torch.equal(a, b) for a, b in zip(got, again))
    f, kw["dx2"] = s["f"].clone(), None if dx2 is None else dx2.clone()
    dx_, df_ = ops.block_norm_bwd(dy, s["x"], f, s["w_pre"], None, **kw, dx=kw["dx2"], df=f)
    assert torch.equal(dx, dx_) and torch.equal(df, df_) and df_ is f
    assert lib.poll_status().wait_giveups == 0


@pytest.mark.gpu
def test_gradient_against_differences(ops):
    """Central differences of the 64-bit forward pass along random directions: step h = 1e-4 leaves h^2 times a third
    derivative (order 1 here), 1e-8, and 1e-12 of cancellation; the fp32 gradients bring 1e-5."""
    s, r = inputs((2, 24, 12), torch.float32, True, "sequence", seed=3)
    dy, dx2 = r(2, 24, 12), r(2, 24, 12)
    base = [t.double() for t in (s["x"], s["f"], s["w_pre"], s["w_post"], s["gate"])]

    def loss(x, f, w_pre, w_post, gate):
        x2 = forward64(x, f, w_post, gate, 0.35)
        return float((norm64(x2, w_pre) * dy.double()).sum() + (x2 * dx2.double()).sum())
    x2 = forward64(*base[:2], base[3], base[4], 0.35).float()
    acc = [torch.zeros(24, device="cuda"), torch.zeros(24, device="cuda"), torch.zeros(2, 24, device="cuda")]
    dx, df = ops.block_norm_bwd(dy, x2, s["f"], s["w_pre"], acc[0], w_post=s["w_post"], dw_post=acc[1], gate=s["gate"], dgate=acc[2], dx2=dx2, alpha=0.35, eps=EPS)
    for k, grad in enumerate((dx, df, acc[0], acc[1], acc[2])):
        d = torch.randn_like(base[k])
        moved = [[t + sign * 1e-4 * d if i == k else t for i, t in enumerate(base)] for sign in (1, -1)]
        slope, dot = (loss(*moved[0]) - loss(*moved[1])) / 2e-4, float((grad.double() * d).sum())
        assert abs(slope - dot) <= 3e-5 * float((grad.double() * d).abs().sum()) + 1e-5, k


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 1024, 64), (2, 100, 33)])
def test_zero_rows_and_a_token_that_is_not_finite(ops, shape):
    """A token whose branch is all zeros keeps its x; NaN and infinity stay in their token."""
    s, _ = inputs(shape, torch.bfloat16, True, "channel")
    s["f"][:, :, 1] = 0
    s["f"][1, 3, 5] = float("nan")
    s["f"][0, 4, 7] = float("inf")
    x2, y = ops.block_norm(s["x"], s["f"], s["w_pre"], w_post=s["w_post"], gate=s["gate"], alpha=0.35, eps=EPS)
    assert torch.equal(x2[:, :, 1], s["x"][:, :, 1])
    bad = torch.zeros(shape[0], shape[2], dtype=torch.bool, device="cuda")
    bad[1, 5] = bad[0, 7] = True
    assert bool(y.isfinite().all(1)[~bad].all()) and not bool(y.isfinite().all(1)[bad].any())


@pytest.mark.gpu
def test_sum_that_cancels(ops):
    """x2 far smaller than x and the branch: its statistics come from x2 itself."""
    s, _ = inputs((1, 512, 64), torch.float32, True, "none")
    branch = forward64(torch.zeros_like(s["f"]), s["f"], s["w_post"], None, 1.0)
    x = (-branch * (1 + 1e-3)).float()
    x2, y = ops.block_norm(x, s["f"], s["w_pre"], w_post=s["w_post"], alpha=1.0, eps=1e-12)
    assert within(y, norm64(x2, s["w_pre"], 1e-12), torch.float32)[0]


@pytest.mark.gpu
def test_captured_and_on_another_stream(ops):
    s, r = inputs((4, 256, 64), torch.bfloat16, True, "sequence")
    dy = r(4, 256, 64, dtype=torch.bfloat16)
    acc = [torch.zeros(256, device="cuda"), torch.zeros(256, device="cuda"), torch.zeros(4, 256, device="cuda")]

    def step(acc):
        x2, y = ops.block_norm(s["x"], s["f"], s["w_pre"], w_post=s["w_post"], gate=s["gate"], alpha=0.35)
        return [x2, y, *ops.block_norm_bwd(dy, x2, s["f"], s["w_pre"], acc[0], w_post=s["w_post"], dw_post=acc[1], gate=s["gate"], dgate=acc[2], alpha=0.35)]
    ref = step(acc)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    other = [torch.zeros_like(t) for t in acc]
    with torch.cuda.graph(graph, stream=stream):
        out = step(other)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref + acc, out + other))


@pytest.mark.gpu
def test_refusals(ops):
    t = [torch.zeros(2, 8, 4, device="cuda") for _ in range(4)]
    w = torch.ones(8, device="cuda")
    with pytest.raises(lib.AneCudaError):
        dev_ops.block_norm(t[0], t[1], w, x2=t[1])
    with pytest.raises(lib.AneCudaError):
        dev_ops.block_norm(t[0], t[1], w, y=t[0])
    with pytest.raises(lib.AneCudaError):
        dev_ops.block_norm_bwd(t[0], t[1], t[2], w, None, dx=t[3], df=t[3])
    with pytest.raises(ValueError):
        dev_ops.block_norm(t[0].transpose(1, 2).contiguous().transpose(1, 2), t[1], w)
    p = [a.data_ptr() for a in t]
    L = lib.load()
    assert L.ane_cuda_block_norm_dev(None, 0, 2, 8, 4, p[0], p[1], p[2], p[3], None, None, 1, w.data_ptr(), 1.0, 1e-5) == lib.ERR_INVALID   # no gate
    assert L.ane_cuda_block_norm_dev(None, 5, 2, 8, 4, p[0], p[1], p[2], p[3], None, None, 0, w.data_ptr(), 1.0, 1e-5) == lib.ERR_INVALID
    assert L.ane_cuda_block_norm_dev(None, 0, 2, 0, 4, p[0], p[1], p[2], p[3], None, None, 0, w.data_ptr(), 1.0, 1e-5) == lib.ERR_INVALID
    lib.set_tuning("check_extents", 1)
    try:
        assert L.ane_cuda_block_norm_dev(None, 0, 1 << 20, 8, 64, p[0], p[1], p[2], p[3], None, None, 0, w.data_ptr(), 1.0, 1e-5) == lib.ERR_INVALID
    finally:
        lib.clear_tuning("check_extents")

"""The norms around a block, the loss head without logits and the AdamW step over a list of tensors together, as a training
step uses them; their outputs between guard zones; their scratch under captured graphs, a frozen library and refused
allocations; and every kernel that a tuning knob can select.

Tolerances.  The step's parameters and activations are fp32, so every operator brings the 1e-5 of its own tests; errors of an
operator pass through at most three more (norm, branch, norm), each of which amplifies them by no more than a small factor: 1e-4
of a gradient's norm.  Knobs select other kernels for the same sums: fp32 sums in another order, 2e-5 of the largest value, and
one rounding of the storage type more.
"""
import math

import pytest
import torch

from ane_b200 import lib
from tests.test_block_norm import chan, forward64, norm64
from tests.test_guards import Guarded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ane_b200 import dev_ops
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    lib.init(0)
    return dev_ops


B, D, S, V, LAYERS = 2, 64, 40, 300, 2


def make_model(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s, scale=1.0, shift=0.0):
        return torch.randn(s, generator=g, device="cuda") * scale + shift
    p = {"table": r(V, D, scale=1 / math.sqrt(D)), "w_in": r(D, scale=0.1, shift=1.0)}
    for k in range(LAYERS):
        p[f"post{k}"], p[f"pre{k}"], p[f"gate{k}"], p[f"mix{k}"] = r(D, scale=0.1, shift=1.0), r(D, scale=0.1, shift=1.0), r(D, scale=0.3, shift=0.5), r(D, D, scale=1 / math.sqrt(D))
    tokens = torch.randint(0, V, (B, S), generator=g, device="cuda", dtype=torch.int32)
    targets = torch.roll(tokens, -1, 1)
    targets[:, -1] = -1                                   # the last token has no successor
    return p, tokens, targets.contiguous()


def own_step(ops, p, tokens, targets, grads):
    """Forward and backward pass: gather, norm, per layer a product (the block), the norms around it; the loss head.  Adds to
    grads; returns the losses."""
    x = ops.embed_lookup(p["table"], tokens)
    y = ops.rmsnorm(x, p["w_in"])
    xs, ys, fs = [x], [y], []
    for k in range(LAYERS):
        fs.append(torch.matmul(p[f"mix{k}"], ys[-1]))
        x2, y = ops.block_norm(xs[-1], fs[-1], p[f"pre{k}"], w_post=p[f"post{k}"], gate=p[f"gate{k}"], alpha=0.5)
        xs.append(x2)
        ys.append(y)
    loss, dy = ops.linear_cross_entropy(ys[-1], p["table"], targets, d_table=grads["table"])
    dx = None
    for k in reversed(range(LAYERS)):
        dx, df = ops.block_norm_bwd(dy, xs[k + 1], fs[k], p[f"pre{k}"], grads[f"pre{k}"], w_post=p[f"post{k}"], dw_post=grads[f"post{k}"], gate=p[f"gate{k}"],
                                    dgate=grads[f"gate{k}"], dx2=dx, alpha=0.5)
        grads[f"mix{k}"] += torch.einsum("bos,bis->oi", df, ys[k])
        dy = torch.matmul(p[f"mix{k}"].t(), df).contiguous()
    dx = ops.rmsnorm_bwd(dy, xs[0], p["w_in"], grads["w_in"], add=dx, exact=True)
    ops.embed_backward(grads["table"], dx, tokens)
    return loss


def reference_step(p, tokens, targets):
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    x = q["table"][tokens.long()].transpose(1, 2)
    y = norm64(x, q["w_in"])
    for k in range(LAYERS):
        f = q[f"mix{k}"] @ y
        n = f / torch.sqrt((f * f).mean(1, keepdim=True) + 1e-5) * q[f"post{k}"][None, :, None]
        x = x + 0.5 * q[f"gate{k}"][None, :, None] * n
        y = x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5) * q[f"pre{k}"][None, :, None]
    lp = torch.log_softmax(torch.einsum("vd,bds->bvs", q["table"], y), 1)
    ok = targets >= 0
    tok = -lp.gather(1, torch.where(ok, targets, 0).long()[:, None])[:, 0] * ok
    loss = tok.sum(1) / S
    grads = torch.autograd.grad(loss.sum(), list(q.values()))
    return loss.detach(), dict(zip(q, grads))


def test_a_training_step(ops):
    p, tokens, targets = make_model()
    grads = {k: torch.zeros_like(v) for k, v in p.items()}
    ref_loss, ref = reference_step(p, tokens, targets)
    loss = own_step(ops, p, tokens, targets, grads)
    assert float((loss.double() - ref_loss).abs().max()) <= 1e-5 * float(ref_loss.max())
    for k in p:
        assert float((grads[k].double() - ref[k]).norm()) <= 1e-4 * float(ref[k].norm()), k
    # one AdamW step over all of them, moments in 8 bits, clipped; fp32 moments beside it
    norm = sum(float(g.double().square().sum()) for g in grads.values()) ** 0.5
    clip = ops.clip_factor(torch.tensor([norm ** 2], device="cuda"), 1.0)
    names = list(p)
    before = {k: v.double() for k, v in p.items()}
    m, v = ([torch.zeros(p[k].shape, dtype=torch.uint8, device="cuda") for k in names] for _ in range(2))
    ms, vs = ([torch.zeros(-(-p[k].numel() // 256), device="cuda") for k in names] for _ in range(2))
    copies = [torch.zeros(p[k].shape, dtype=torch.bfloat16, device="cuda") for k in names]
    tensors = ops.AdamTensors([p[k] for k in names], [grads[k] for k in names], m, v, m_scale=ms, v_scale=vs, copy=copies, wd=[0.1 if p[k].dim() == 2 else 0.0 for k in names])
    ops.adam_multi(tensors, 1, 1e-3, 0.9, 0.95, 1e-8, clip=clip, seed=1)
    for i, k in enumerate(names):
        g = grads[k].double() * min(1.0, 1.0 / norm)
        want = before[k] - 1e-3 * (g / (g.abs() + 1e-8) + (0.1 if p[k].dim() == 2 else 0.0) * before[k])      # at t = 1 the moments' quotient is the sign
        # where the gradient is no larger than eps the quotient hangs on its rounding; elsewhere five roundings and two approximations
        sure = g.abs() > 1e-6
        assert float(((p[k].double() - want).abs() - 2e-6 * want.abs() - 2e-8)[sure].max()) <= 0, k
        assert torch.equal(copies[i], p[k].bfloat16())
    # the next step runs on the new weights, its products on the 16-bit copy of the table
    x = ops.embed_lookup(copies[0], tokens)
    y = ops.rmsnorm(x, p["w_in"])
    loss16, dx16 = ops.linear_cross_entropy(y, copies[0], targets)
    logits = torch.einsum("vd,bds->bvs", copies[0].double(), y.double())
    ref16 = -torch.log_softmax(logits, 1).gather(1, torch.where(targets >= 0, targets, 0).long()[:, None])[:, 0] * (targets >= 0)
    assert float((loss16.double() - ref16.sum(1) / S).abs().max()) <= 1e-5 * float(ref16.max())
    assert bool(dx16.isfinite().all())


def test_two_captured_steps_share_the_scratch(ops):
    """Graphs of two models whose operators use the same scratch range, replayed in turn, then the library made to grow it."""
    models = [make_model(s) for s in (1, 2)]
    want, graphs, grads = [], [], []
    for p, tokens, targets in models:
        g = {k: torch.zeros_like(v) for k, v in p.items()}
        loss = own_step(ops, p, tokens, targets, g)
        want.append((loss.clone(), {k: v.clone() for k, v in g.items()}))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    losses = []
    for p, tokens, targets in models:
        g = {k: torch.zeros_like(v) for k, v in p.items()}
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            losses.append(own_step(ops, p, tokens, targets, g))
        graphs.append(graph)
        grads.append(g)
    x = torch.randn(1, 64, 2048, device="cuda")           # an eager call with a larger scratch
    ops.linear_cross_entropy(x, torch.randn(20000, 64, device="cuda") / 8, torch.zeros(1, 2048, dtype=torch.int32, device="cuda"))
    for i in (0, 1, 0):
        for g in grads[i].values():
            g.zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(losses[i], want[i][0]), i
        for k in grads[i]:
            if not k.startswith("mix"):                  # torch's own product
                assert torch.equal(grads[i][k], want[i][1][k]), (i, k)


def test_refused_allocations_and_a_frozen_library(ops):
    """A scratch that cannot grow is an error that names the operator, and the next call works."""
    L = lib.load()
    x, t = torch.randn(1, 64, 33, device="cuda"), torch.zeros(1, 33, dtype=torch.int32, device="cuda")
    E = torch.randn(50, 64, device="cuda")
    want = ops.linear_cross_entropy(x, E, t)[0]
    big = L.ane_cuda_workspace_bytes()
    V_big = 4096 * (2 + big // (1 << 20))                  # its dl alone is larger than the scratch there is
    E_big, x_big, t_big = torch.randn(V_big, 8, device="cuda"), torch.randn(1, 8, 2048, device="cuda"), torch.zeros(1, 2048, dtype=torch.int32, device="cuda")
    if 2048 * V_big * 4 < 768 << 20:                       # pieces stop growing there
        lib.check(L.ane_cuda_freeze(1))
        try:
            with pytest.raises(lib.AneCudaError, match="linear_cross_entropy"):
                ops.linear_cross_entropy(x_big, E_big, t_big)
        finally:
            lib.check(L.ane_cuda_freeze(0))
        lib.set_tuning("fail_alloc", 2)
        try:
            with pytest.raises(lib.AneCudaError, match="linear_cross_entropy"):
                ops.linear_cross_entropy(x_big, E_big, t_big)
        finally:
            lib.clear_tuning("fail_alloc")
    assert torch.equal(ops.linear_cross_entropy(x, E, t)[0], want)


KNOBS = [("block_norm_cluster", v) for v in (0, 1, 3, 5)] + [("linear_xent_wide", v) for v in (0, 1)] + [("linear_xent_dep", 0)]


@pytest.mark.parametrize("knob,value", KNOBS)
def test_alternate_kernels(ops, knob, value):
    g = torch.Generator(device="cuda").manual_seed(9)
    lib.poll_status()
    for dt in (torch.float32, torch.bfloat16):
        x, f, dy, dx2 = (torch.randn(24, 512, 520, generator=g, device="cuda").to(dt) for _ in range(4))
        w, v, gate = (torch.randn(512, generator=g, device="cuda") for _ in range(3))
        E, t = (torch.randn(3000, 512, generator=g, device="cuda") / 22).to(dt), torch.randint(0, 3000, (2, 520), generator=g, device="cuda", dtype=torch.int32)

        def everything():
            acc = [torch.zeros(512, device="cuda") for _ in range(3)] + [torch.zeros(3000, 512, device="cuda")]
            x2, y = ops.block_norm(x, f, w, w_post=v, gate=gate, alpha=0.3)
            dx, df = ops.block_norm_bwd(dy, x, f, w, acc[0], w_post=v, dw_post=acc[1], gate=gate, dgate=acc[2], dx2=dx2, alpha=0.3)
            loss, dxe = ops.linear_cross_entropy(x[:2].contiguous(), E, t, d_table=acc[3])
            return [x2, y, dx, df, dxe], acc + [loss]
        want = everything()
        lib.set_tuning(knob, value)
        try:
            got = everything()
        finally:
            lib.clear_tuning(knob)
        for a, b in zip(got[0], want[0]):
            tol = torch.finfo(dt).eps * b.double().abs() + 2e-5 * float(b.abs().max())
            assert bool(((a.double() - b.double()).abs() <= tol).all())
        for a, b in zip(got[1], want[1]):
            assert float((a - b).norm()) <= 2e-5 * float(b.norm()) + 1e-6
    assert lib.poll_status().wait_giveups == 0


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(3, 7, 5), (2, 1000, 33), (2, 129, 264), (24, 256, 520), (2, 2048, 72), (1, 4000, 24), (70, 128, 8)])
def test_block_norm_stays_inside_its_outputs(ops, shape, dt):
    Bn, C, Sn = shape
    g = torch.Generator(device="cuda").manual_seed(2)
    x, f, dy, dx2 = (torch.randn(*shape, generator=g, device="cuda").to(dt) for _ in range(4))
    w, v, gate = torch.randn(C, device="cuda"), torch.randn(C, device="cuda"), torch.randn(Bn, C, device="cuda")
    G = Guarded(torch)
    for knob in (0, 1, 3, 7):
        lib.set_tuning("block_norm_cluster", knob)
        try:
            ops.block_norm(x, f, w, w_post=v, gate=gate, alpha=0.3, x2=G.new(shape, dt), y=G.new(shape, dt))
            ops.block_norm_bwd(dy, x, f, w, G.new((C,), torch.float32, fill=0.0), w_post=v, dw_post=G.new((C,), torch.float32, fill=0.0), gate=gate,
                               dgate=G.new((Bn, C), torch.float32, fill=0.0), dx2=dx2, alpha=0.3, dx=G.new(shape, dt), df=G.new(shape, dt))
            G.check(f"block_norm, knob {knob}")
        finally:
            lib.clear_tuning("block_norm_cluster")
    # outputs off a 16-byte boundary
    ops.block_norm(x, f, w, w_post=v, gate=gate, alpha=0.3, x2=G.new(shape, dt, misalign=1), y=G.new(shape, dt, misalign=3))
    G.check("block_norm, misaligned")


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B_,D_,V_,S_", [(1, 5, 7, 3), (3, 100, 1001, 77), (2, 256, 513, 264), (1, 300, 5000, 130)])
def test_linear_cross_entropy_stays_inside_its_outputs(ops, B_, D_, V_, S_, dt):
    g = torch.Generator(device="cuda").manual_seed(3)
    x, E = torch.randn(B_, D_, S_, generator=g, device="cuda").to(dt), torch.randn(V_, D_, generator=g, device="cuda").to(dt)
    t = torch.randint(-1, V_ + 1, (B_, S_), generator=g, device="cuda", dtype=torch.int32)
    G = Guarded(torch)
    for knobs in ((), (("linear_xent_wide", 0),), (("linear_xent_wide", 1),)):
        for k, v in knobs:
            lib.set_tuning(k, v)
        try:
            ops.linear_cross_entropy(x, E, t, d_table=G.new((V_, D_), torch.float32, fill=0.0), dx=G.new((B_, D_, S_), dt), loss_tok=G.new((B_, S_), torch.float32))
            G.check(f"linear_cross_entropy {knobs}")
        finally:
            for k, _ in knobs:
                lib.clear_tuning(k)


@pytest.mark.parametrize("mis", [0, 1])
@pytest.mark.parametrize("n", [1, 255, 256, 257, 5000])
def test_adam_multi_stays_inside_its_outputs(ops, n, mis):
    G = Guarded(torch)
    g = torch.randn(n, device="cuda")
    blocks = -(-n // 256)
    for q8 in (False, True):
        w, copy = G.new((n,), torch.float32, fill=0.5, misalign=mis), G.new((n,), torch.bfloat16, misalign=mis)
        if q8:
            m, v = (G.new((n,), torch.uint8, fill=0, misalign=mis) for _ in range(2))
            s = [[G.new((blocks,), torch.float32, fill=0.0)] for _ in range(2)]
        else:
            m, v = (G.new((n,), torch.float32, fill=0.0, misalign=mis) for _ in range(2))
            s = [None, None]
        ops.adam_multi(ops.AdamTensors([w], [g], [m], [v], *s, copy=[copy]), 1, 1e-3, 0.9, 0.95, 1e-8)
        if q8:
            ops.adam_state_unpack(m, s[0][0], out=G.new((n,), torch.float32, misalign=mis))
            ops.adam_state_pack(g, codes=G.new((n,), torch.uint8, misalign=mis), scales=G.new((blocks,), torch.float32))
        G.check(f"adam_multi, 8 bits {q8}")


def test_forward64_is_the_formula_the_step_uses():
    """The two references of this file and of the operator's own tests agree."""
    x, f = torch.randn(1, 8, 3, device="cuda"), torch.randn(1, 8, 3, device="cuda")
    n = f.double() / torch.sqrt((f.double() ** 2).mean(1, keepdim=True) + 1e-5)
    assert torch.allclose(forward64(x, f, torch.ones(8, device="cuda"), None, 0.5), x.double() + 0.5 * n) and chan(None) == 1.0

"""Classifier product and cross-entropy without the logits (linear_cross_entropy) against 64-bit formulas, autograd,
differences and the operator over given logits.

Tolerances, as the 2-norm of the difference over that of the result, and as the largest difference over the largest value.
A logit is an fp32 sum of D products: its error is below about sqrt(D) * 2^-24 of the norm of its terms, 2e-6 for D = 1000;
fp32 inputs enter as two 16-bit parts, which drops low * low and rounds the low part: 2^-17 = 7.6e-6 of a term at most (bf16
parts; fp16 ones, scaled, 2^-21), random in sign, so of the norm of the terms.  Logits here are of order 1 (up to 6 where scaled up), so
probabilities carry a relative error of at most about 1e-5, and the loss, a mean of numbers of order log V, less.
  loss                1e-5
  d_table, fp32       dl in two parts leaves 2^-16 of it (bf16) in the worst case, half a step of the second rounding of
                      half a step, random: 2-norm 1e-5 with the above; largest value 3e-5
  dx, fp32            the same
  dx, 16 bits         dl rounded once (half a step, relative: 2^-9 / sqrt 3 on average for bf16, at most 2^-8 in the norm) and
                      the result rounded once: 2 * eps/2 + 1e-5 in the 2-norm, 2.1 * eps/2 of the largest value
"""
import math

import pytest
import torch

from ane_b200 import dev_ops, lib

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def reference(x, table, targets, grad_scale=1.0):
    """loss_seq, loss_tok, dx, dE in 64 bits."""
    B, D, S = x.shape
    X, E = x.double(), table.double()
    y = targets.long() if targets.dtype != torch.uint16 else targets.to(torch.int32).long()
    ok = (y >= 0) & (y < E.shape[0])
    at = torch.where(ok, y, 0)[:, None, :]
    X = torch.where(ok[:, None, :], X, torch.zeros_like(X))           # a token without a target is not looked at
    logits = torch.einsum("vd,bds->bvs", E, X)
    lp = torch.log_softmax(logits, 1)
    tok = torch.where(ok, -torch.log(torch.exp(lp.gather(1, at)[:, 0]) + 1e-10), torch.zeros_like(lp[:, 0]))
    dl = lp.exp().scatter_add(1, at, -torch.ones_like(at, dtype=torch.float64)) * ok[:, None, :] * (grad_scale / S)
    return tok.sum(1) / S, tok, torch.einsum("vd,bvs->bds", E, dl), torch.einsum("bvs,bds->vd", dl, X)


def off(got, ref, part=0.0):
    """`part`: the size of the numbers whose difference a value is, below which errors do not shrink (probability 1 less
    the one of the target; the sum 1 + 1e-10 in a loss)."""
    d, ref = got.double() - ref.double(), ref.double()
    return float(d.norm() / max(float(ref.norm()), part)), float(d.abs().max() / max(float(ref.abs().max()), part))


def check_grads(dt, dx, dx_ref, dE=None, dE_ref=None, part_x=0.0, part_E=0.0):
    half = torch.finfo(dt).eps / 2
    two, most = off(dx, dx_ref, part_x)
    if dt == torch.float32:
        assert two <= 1e-5 and most <= 3e-5, (two, most)
    else:
        assert two <= 2 * half + 1e-5 and most <= 2.1 * half, (two, most)
    if dE is not None:
        two, most = off(dE, dE_ref, part_E)
        assert two <= 1e-5 and most <= 3e-5, (two, most)


# ------------------------------------------------------------------ CPU
def test_refusals_without_a_gpu():
    x, E, t = torch.zeros(2, 8, 4), torch.zeros(10, 8), torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="table"):
        dev_ops.linear_cross_entropy(x, torch.zeros(10, 9), t)
    with pytest.raises(ValueError, match="table"):
        dev_ops.linear_cross_entropy(x, E.bfloat16(), t)
    with pytest.raises(ValueError, match="targets"):
        dev_ops.linear_cross_entropy(x, E, t.long())
    with pytest.raises(ValueError, match="targets"):
        dev_ops.linear_cross_entropy(x, E, t[:, :3])
    with pytest.raises(ValueError, match="d_table"):
        dev_ops.linear_cross_entropy(x, E, t, d_table=torch.zeros(10, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="losses alone"):
        dev_ops.linear_cross_entropy(x, E, t, grad=False, d_table=torch.zeros(10, 8))
    with pytest.raises(ValueError, match="loss_tok"):
        dev_ops.linear_cross_entropy(x, E, t, loss_tok=torch.zeros(2, 5))
    with pytest.raises(ValueError, match="current CUDA device"):
        dev_ops.linear_cross_entropy(x, E, t)


def test_the_library_refuses_before_init():
    if torch.cuda.is_available():
        return
    assert lib.load().ane_cuda_linear_cross_entropy_dev(None, 0, 1, 1, 1, 1, 1, *[None] * 7, 1.0) == lib.ERR_NOT_INIT


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    lib.init(0)
    lib.poll_status()
    yield dev_ops
    assert lib.poll_status().wait_giveups == 0


def inputs(B, D, V, S, dt, seed=0, scale=1.0, masked=0.1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(B, D, S, generator=g, device="cuda").to(dt)
    E = (torch.randn(V, D, generator=g, device="cuda") * scale / math.sqrt(D)).to(dt)
    t = torch.randint(0, V, (B, S), generator=g, device="cuda", dtype=torch.int32)
    t[torch.rand(B, S, generator=g, device="cuda") < masked] = -1
    return x, E, t


# tiles of 128 tokens and 256 rows, K blocks of 64: one below, at and above them; rows that break alignment; several pieces
SHAPES = [(1, 8, 1, 1), (1, 64, 256, 128), (2, 64, 255, 1), (1, 72, 257, 129), (3, 33, 100, 5), (1, 1, 2, 3), (2, 200, 1000, 77), (1, 768, 9200, 256),
          (5, 130, 513, 200), (1, 256, 20000, 16), (2, 96, 5000, 1100),
          (1, 256, 777, 4), (2, 64, 1001, 2), (4, 136, 300, 1), (1, 1709, 478, 1), (1, 1032, 2000, 1), (1, 96, 5, 2)]      # one to four tokens


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_losses_and_gradients(ops, shape, dt):
    B, D, V, S = shape
    x, E, t = inputs(B, D, V, S, DT[dt])
    t[0, 0] = V - 1
    before = torch.randn(V, D, device="cuda") * 1e-6
    dE, tok = before.clone(), torch.full((B, S), -7.0, device="cuda")
    loss, dx = ops.linear_cross_entropy(x, E, t, d_table=dE, grad_scale=0.7, loss_tok=tok)
    ref = reference(x, E, t, 0.7)
    assert max(off(loss, ref[0], 0.1)) <= 1e-5 and max(off(tok, ref[1], 0.1)) <= 1e-5, (off(loss, ref[0]), off(tok, ref[1]))
    check_grads(DT[dt], dx, ref[2], dE, ref[3] + before.double(), 0.7 / S * float(E.abs().max()), 0.7 / S * float(x.abs().max()))
    # each gradient alone, and the losses alone: the same bits
    dE2 = before.clone()
    loss2, dx2 = ops.linear_cross_entropy(x, E, t, grad_scale=0.7)
    assert torch.equal(loss, loss2) and torch.equal(dx, dx2)
    L = lib.load()
    rc = L.ane_cuda_linear_cross_entropy_dev(torch.cuda.current_stream().cuda_stream, dev_ops._dt(x), lib.ID_I32, B, D, V, S, loss2.data_ptr(), None, None,
                                             dE2.data_ptr(), x.data_ptr(), E.data_ptr(), t.data_ptr(), 0.7)
    assert rc == lib.OK and torch.equal(dE, dE2)
    assert torch.equal(ops.linear_cross_entropy(x, E, t, grad=False)[0], loss)


@pytest.mark.gpu
@pytest.mark.parametrize("knob", [("linear_xent_few", 0), ("linear_xent_wide", 0), ("linear_xent_wide", 1), ("linear_xent_narrow", 0), ("linear_xent_narrow", 1), ("linear_xent_dep", 0)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1, 64, 700, 1), (3, 33, 100, 1), (2, 200, 1300, 77), (1, 520, 600, 300)])
def test_alternate_kernels(ops, shape, dt, knob):
    B, D, V, S = shape
    x, E, t = inputs(B, D, V, S, DT[dt], seed=10)
    t[0, 0] = 0
    dE = torch.zeros(V, D, device="cuda")
    lib.set_tuning(*knob)
    try:
        loss, dx = ops.linear_cross_entropy(x, E, t, d_table=dE)
    finally:
        lib.clear_tuning(knob[0])
    ref = reference(x, E, t)
    assert max(off(loss, ref[0])) <= 1e-5
    check_grads(DT[dt], dx, ref[2], dE, ref[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_more_tokens_than_one_round(ops, dt):
    """8192 tokens are one round: d_table grows over several, the last of them short."""
    x, E, t = inputs(17, 64, 700, 1000, DT[dt], seed=1)
    dE, tok = torch.zeros(700, 64, device="cuda"), torch.zeros(17, 1000, device="cuda")
    loss, dx = ops.linear_cross_entropy(x, E, t, d_table=dE, loss_tok=tok)
    ref = reference(x, E, t)
    assert max(off(loss, ref[0])) <= 1e-5 and max(off(tok, ref[1])) <= 1e-5
    check_grads(DT[dt], dx, ref[2], dE, ref[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dt,D,V", [("f32", 1024, 70000), ("f16", 1001, 140000)])
def test_a_table_that_is_packed_piece_by_piece(ops, dt, D, V):
    x, E, t = inputs(2, D, V, 130, DT[dt], seed=12)                # more than 256 MiB of packed rows
    dE = torch.zeros(V, D, device="cuda")
    loss, dx = ops.linear_cross_entropy(x, E, t, d_table=dE)
    ref = reference(x, E, t)
    assert max(off(loss, ref[0])) <= 1e-5
    check_grads(DT[dt], dx, ref[2], dE, ref[3])
    alone, _ = ops.linear_cross_entropy(x, E, t, grad=False)
    assert max(off(alone, ref[0])) <= 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(40, 64, 300, 7), (300, 64, 300, 1), (8, 64, 300, 40)])
def test_many_short_sequences(ops, shape, dt):
    x, E, t = inputs(*shape, DT[dt], seed=13)
    loss, dx = ops.linear_cross_entropy(x, E, t)
    ref = reference(x, E, t)
    assert max(off(loss, ref[0])) <= 1e-5
    check_grads(DT[dt], dx, ref[2])
    alone, _ = ops.linear_cross_entropy(x, E, t, grad=False)
    assert torch.equal(alone, loss)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_offset_views_and_uint16_targets(ops, dt):
    """A table that starts off a 16-byte boundary, and the id type of the reference."""
    dt = DT[dt]
    x, E, t = inputs(2, 64, 600, 40, dt, seed=2, masked=0.0)
    raw = torch.zeros(600 * 64 + 1, dtype=dt, device="cuda")
    odd = raw[1:].view(600, 64)
    odd.copy_(E)
    t16 = t.to(torch.int32)
    t16[1, 7] = 65535                                                  # no such row
    ids = t16.to(torch.int16).view(torch.uint16) if hasattr(torch, "uint16") else t16.to(torch.int16)
    dE, dE2 = torch.zeros(600, 64, device="cuda"), torch.zeros(600, 64, device="cuda")
    lib.poll_status()
    loss, dx = ops.linear_cross_entropy(x, odd, ids, d_table=dE)
    assert lib.poll_status().oor_ids == 1
    t[1, 7] = -1
    loss2, dx2 = ops.linear_cross_entropy(x, E, t, d_table=dE2)
    assert lib.poll_status().oor_ids == 0
    assert torch.equal(loss, loss2) and torch.equal(dx, dx2) and torch.equal(dE, dE2)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_masked_tokens_hide_what_they_hold(ops, dt):
    x, E, t = inputs(2, 64, 700, 300, DT[dt], seed=3, masked=0.0)
    t[0, 17] = t[1, 299] = -100
    t[1, :128] = -1                                                    # a whole tile of tokens
    x[0, :, 17], x[1, 3, 299], x[1, :, 5] = float("nan"), float("inf"), -float("inf")
    dE, tok = torch.zeros(700, 64, device="cuda"), torch.ones(2, 300, device="cuda")
    loss, dx = ops.linear_cross_entropy(x, E, t, d_table=dE, loss_tok=tok)
    ref = reference(torch.where(t[:, None, :] < 0, torch.zeros_like(x), x), E, t)
    assert max(off(loss, ref[0])) <= 1e-5
    check_grads(DT[dt], dx, ref[2], dE, ref[3])
    assert bool((dx.transpose(1, 2)[t < 0] == 0).all()) and bool((tok[t < 0] == 0).all())
    t[:] = -1
    dE.zero_()
    loss, dx = ops.linear_cross_entropy(x, E, t, d_table=dE)
    assert not bool(loss.any()) and not bool(dx.any()) and not bool(dE.any())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 40, 300, 1), (1, 40, 300, 3), (2, 40, 300, 50)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_a_table_that_is_not_finite_leaves_masked_tokens_alone(ops, dt, shape):
    x, E, t = inputs(*shape, DT[dt], 9, masked=0.0)
    E[7, 3], E[90, 20] = float("inf"), float("nan")
    t[0, 0] = -1
    tok = torch.ones(t.shape, device="cuda")
    _, dx = ops.linear_cross_entropy(x, E, t, loss_tok=tok)
    assert float(tok[0, 0]) == 0 and not dx[0, :, 0].float().any()
    lib.poll_status()


@pytest.mark.gpu
def test_a_token_that_is_not_finite_shows_and_is_counted(ops):
    x, E, t = inputs(1, 64, 700, 200, torch.bfloat16, seed=4, masked=0.0)
    x[0, 5, 9] = float("nan")
    tok = torch.zeros(1, 200, device="cuda")
    lib.poll_status()
    loss, _ = ops.linear_cross_entropy(x, E, t, grad=False, loss_tok=tok)
    assert bool(loss.isnan().all()) and lib.poll_status().nonfinite == 1
    assert bool(tok[0, 9].isnan()) and bool(tok[0, torch.arange(200) != 9].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_large_logits(ops, dt):
    """Logits of up to several hundred, of one sign and mixed: the running maximum carries them.  A logit's error grows with it:
    of a term's 7.6e-6, times 40 (the terms' norm)."""
    x, E, t = inputs(1, 128, 3000, 130, DT[dt], seed=5, scale=40.0)
    tok = torch.zeros(1, 130, device="cuda")
    loss, dx = ops.linear_cross_entropy(x, E, t, loss_tok=tok)
    ref = reference(x, E, t)
    live = ref[1] < 22.0                                               # above, log(p + 1e-10) saturates at 23.03
    assert float((tok.double() - ref[1])[live].abs().max()) <= 40 * 7.6e-6 * 3 and float(tok.max()) <= 23.03
    assert off(dx, ref[2])[0] <= 2 * torch.finfo(DT[dt]).eps / 2 + 40 * 7.6e-6 * 3
    loss, _ = ops.linear_cross_entropy(x.abs(), -E.abs(), t, grad=False)
    assert abs(float(loss[0]) - float(reference(x.abs(), -E.abs(), t)[0][0])) <= 2e-3


@pytest.mark.gpu
def test_agrees_with_the_operator_over_given_logits(ops):
    """The same loss and the same gradient of the logits as cross_entropy over fp32 logits."""
    x, E, t = inputs(2, 64, 1000, 64, torch.float32, seed=6, masked=0.0)
    logits = torch.einsum("vd,bds->bvs", E.double(), x.double()).float().contiguous()
    loss, dl = ops.cross_entropy(logits, t, grad_scale=0.5)
    dE = torch.zeros(1000, 64, device="cuda")
    loss2, dx = ops.linear_cross_entropy(x, E, t, d_table=dE, grad_scale=0.5)
    assert max(off(loss2, loss)) <= 1.5e-5
    check_grads(torch.float32, dx, torch.einsum("vd,bvs->bds", E.double(), dl.double()), dE, torch.einsum("bvs,bds->vd", dl.double(), x.double()))


@pytest.mark.gpu
def test_gradients_against_differences(ops):
    """Central differences of the 64-bit loss: step 1e-4, 1e-8 of curvature; the gradients bring 1e-5 of theirs."""
    x, E, t = inputs(1, 16, 50, 20, torch.float32, seed=7)
    dE = torch.zeros(50, 16, device="cuda")
    _, dx = ops.linear_cross_entropy(x, E, t, d_table=dE)
    for k, grad in enumerate((dx, dE)):
        base = [x.double(), E.double()]
        d = torch.randn_like(base[k])
        moved = [[b + s * 1e-4 * d if i == k else b for i, b in enumerate(base)] for s in (1, -1)]
        slope = float(reference(*moved[0], t)[0].sum() - reference(*moved[1], t)[0].sum()) / 2e-4
        assert abs(slope - float((grad.double() * d).sum())) <= 3e-5 * float((grad.double() * d).abs().sum()) + 1e-7


@pytest.mark.gpu
def test_repeats_bit_for_bit_captured_and_on_another_stream(ops):
    x, E, t = inputs(2, 128, 3000, 150, torch.bfloat16, seed=8)
    dE = [torch.zeros(3000, 128, device="cuda") for _ in range(2)]
    ref = ops.linear_cross_entropy(x, E, t, d_table=dE[0])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out = ops.linear_cross_entropy(x, E, t, d_table=dE[1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(ref[0], out[0]) and torch.equal(ref[1], out[1]) and torch.equal(*dE)


@pytest.mark.gpu
def test_refusals(ops):
    x, E, t = inputs(1, 8, 10, 4, torch.float32)
    loss = torch.zeros(1, device="cuda")
    L = lib.load()

    def call(dt=0, idt=1, B=1, D=8, V=10, S=4, loss_p=loss.data_ptr(), dx=None, xp=x.data_ptr()):
        return L.ane_cuda_linear_cross_entropy_dev(None, dt, idt, B, D, V, S, loss_p, None, dx, None, xp, E.data_ptr(), t.data_ptr(), 1.0)
    assert call() == lib.OK
    for bad in (dict(dt=3), dict(idt=2), dict(B=0), dict(D=0), dict(V=0), dict(S=0), dict(loss_p=None), dict(xp=None), dict(dx=x.data_ptr()), dict(D=70000),
                dict(B=1 << 20, S=1 << 20), dict(B=(1 << 30) + 1, S=1), dict(V=(1 << 30) + 1), dict(V=(1 << 31) - 257)):
        assert call(**bad) == lib.ERR_INVALID, bad
    lib.set_tuning("check_extents", 1)
    try:
        assert call(V=1 << 28) == lib.ERR_INVALID
    finally:
        lib.clear_tuning("check_extents")
    torch.cuda.synchronize()

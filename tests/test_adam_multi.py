"""The AdamW step over a list of tensors (adam_multi) and the conversion of 8-bit moments.

References: the update in 64-bit numpy; the codes of 8-bit moments in numpy fp32 (the encoding is defined on fp32 values, so
codes are compared exactly); the code tables by enumerating the 256 codes.
Tolerances.  fp32 results: each of m, v takes at most four roundings of 2^-24 relative to terms that do not exceed the sum of
magnitudes, and w adds a square root, two divisions, three products and a sum: 16 * 2^-24 = 9.5e-7 of max(|w|, lr-sized update)
bounds them; 2e-6 is used.  A 16-bit copy is one rounding of w: 2^-8 (bf16) or 2^-11 (fp16) of it.
"""
import numpy as np
import pytest
import torch

from ane_b200 import dev_ops, lib

BLOCK = 256
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HYPER = dict(t=7, lr=1e-2, b1=0.9, b2=0.95, eps=1e-8)


# ------------------------------------------------------------------ references
def values_of_codes(second):
    """The 256 values that codes stand for before the scale, from their fields."""
    out = []
    for c in range(256):
        bits, bias, sign = (5, 15, 1.0) if second else (4, 7, -1.0 if c >= 128 else 1.0)
        e, f = (c >> 3) & ((1 << bits) - 1), (c & 7) / 8.0
        out.append(sign * ((1 + f) * 2.0 ** (e - bias) if e else f * 2.0 ** (1 - bias)))
    return np.array(out)


def decode(codes, scales, second):
    table = values_of_codes(second).astype(np.float32)
    n = codes.size
    return table[codes] * np.repeat(scales, BLOCK)[:n]


def mix(h):
    h = (h ^ (h >> np.uint64(16))) * np.uint64(0x85EBCA6B) & np.uint64(0xFFFFFFFF)
    h = (h ^ (h >> np.uint64(13))) * np.uint64(0xC2B2AE35) & np.uint64(0xFFFFFFFF)
    return h ^ (h >> np.uint64(16))


def noise(n, seed, index, second):
    key = mix(np.uint64((seed + 0x9E3779B9 * index) & 0xFFFFFFFF))
    h = mix((np.arange(n, dtype=np.uint64) * np.uint64(0x9E3779B1) + key) & np.uint64(0xFFFFFFFF))
    return (h & np.uint64(0xFFFFF) if second else h >> np.uint64(12)).astype(np.int64)


def encode(value, seed, index, second):
    """fp32 values -> (codes, scales) exactly as the operator defines them."""
    n, top = value.size, np.float32(122880.0 if second else 480.0)
    v = np.zeros(-(-n // BLOCK) * BLOCK, np.float32)
    v[:n] = value
    most = np.abs(v).reshape(-1, BLOCK).max(1)
    most = np.where(most < np.float32(2.0 ** -100), np.float32(0), most)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        inv = np.where(most > 0, (np.float32(1) / most) * top, np.float32(0)).astype(np.float32)
    y = (np.abs(v) * np.repeat(inv, BLOCK)) * np.float32(2.0 ** (-112 if second else -120))
    r = np.zeros(v.size, np.int64)
    r[:n] = noise(n, seed, index, second)
    c = np.minimum((y.view(np.int32).astype(np.int64) + r) >> 20, 255 if second else 127)
    c = np.where((c == 0) & (y > 0), 1, c) if second else np.where(v < 0, c + 128, c)
    return c[:n].astype(np.uint8), (most * (np.float32(1) / top)).astype(np.float32)


def moments32(g, m, v, b1, b2, gscale, clip):
    """The new moments in fp32, in the operator's order of operations."""
    f = np.float32
    g = g.astype(f) * f(gscale) * f(clip)
    m = f(b1) * m + (f(1) - f(b1)) * g
    return m, f(b2) * v + ((f(1) - f(b2)) * g) * g


def update64(w, g, m, v, t, lr, b1, b2, eps, wd, gscale, clip, dynamic):
    b1f, b2f = float(np.float32(b1)), float(np.float32(b2))
    g = g.astype(np.float64) * gscale * clip
    m, v = b1f * m + (1 - b1f) * g, b2f * v + (1 - b2f) * g * g
    step = m / (1 - b1f ** t) / (np.sqrt(v / (1 - b2f ** t)) + eps)
    return w - lr * (step + wd * w if dynamic else step), m, v


# ------------------------------------------------------------------ CPU: tables, refusals
def test_code_tables_are_monotonic_and_cover_the_stated_range():
    first, second = values_of_codes(False), values_of_codes(True)
    assert first[127] == 480.0 and second[255] == 122880.0
    assert (np.diff(first[:128]) > 0).all() and (np.diff(second) > 0).all()
    assert (first[128:] == -first[:128]).all()
    assert first[1] == 2.0 ** -9 and second[1] == 2.0 ** -17


def test_rounding_keeps_the_mean():
    """Over all 2^20 noise values the mean of the rounded value is the value: exact by construction within a binade; checked
    for a few values against the mean over the hash's noise, whose standard error is spacing / 2 / sqrt(n)."""
    table = values_of_codes(True)
    for x in (0.3, 1.0, 77.7, 3.1e4, 1e-4):
        n = 1 << 16
        v = np.full(n, np.float32(x), np.float32)
        y = v * np.float32(2.0 ** -112)
        c = (y.view(np.int32).astype(np.int64) + noise(n, 5, 0, True)) >> 20
        spacing = table[c.max()] - table[c.min()]
        assert abs(table[c].mean() - x) <= 5 * max(spacing, 1e-9) / 2 / np.sqrt(n) + 1e-6 * x


def test_refusals_without_a_gpu():
    f = [torch.zeros(4)]
    with pytest.raises(ValueError, match="g: expected 1"):
        dev_ops.AdamTensors(f, [], f, f)
    with pytest.raises(ValueError, match="belong to uint8"):
        dev_ops.AdamTensors(f, f, [torch.zeros(4, dtype=torch.uint8)], f)
    with pytest.raises(ValueError, match=r"m\[0\]"):
        dev_ops.AdamTensors(f, f, [torch.zeros(5)], f)
    with pytest.raises(ValueError, match="bf16 or fp16"):
        dev_ops.AdamTensors(f, [torch.zeros(4)], [torch.zeros(4)], [torch.zeros(4)], copy=[torch.zeros(4)])
    with pytest.raises(ValueError, match="share memory"):
        dev_ops.AdamTensors(f, [torch.zeros(4)], [torch.zeros(4)], f)
    with pytest.raises(ValueError, match="current CUDA device"):
        dev_ops.AdamTensors(f, [torch.zeros(4)], [torch.zeros(4)], [torch.zeros(4)])
    with pytest.raises(ValueError, match="scales"):
        dev_ops.adam_state_unpack(torch.zeros(257, dtype=torch.uint8), torch.zeros(1), out=torch.zeros(257))


def test_a_gradient_in_memory_that_the_step_writes_is_refused():
    w, m, v = torch.zeros(1, 8).unbind(0), [torch.zeros(8)], [torch.zeros(8)]
    for g in (w, m, [torch.empty(0).set_(v[0].untyped_storage(), 4, (4,))]):
        a = 4 if g[0].numel() == 4 else 8
        with pytest.raises(ValueError, match="share memory"):
            dev_ops.AdamTensors([t[:a] for t in w], list(g), [t[:a] for t in m], [t[-a:] for t in v])
    g = torch.zeros(8)                    # two weights with one gradient: only read, and so refused for being on the CPU alone
    with pytest.raises(ValueError, match="current CUDA device"):
        dev_ops.AdamTensors([torch.zeros(8), torch.zeros(8)], [g, g], *[[torch.zeros(8), torch.zeros(8)] for _ in range(2)])


def test_the_library_refuses_before_init():
    if torch.cuda.is_available():
        return
    L = lib.load()
    assert L.ane_cuda_adam_multi_dev(None, 0, 0, 1, 0, None, 1, 1.0, 0.9, 0.9, 0.0, 1.0, None, 0, 0) == lib.ERR_NOT_INIT
    assert L.ane_cuda_adam_state_unpack_dev(None, 0, None, None, None, 0) == lib.ERR_NOT_INIT
    assert L.ane_cuda_adam_state_pack_dev(None, 0, None, None, None, 0, 0) == lib.ERR_NOT_INIT


# ------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    lib.init(0)
    return dev_ops


def make(rng, sizes, gdt, offset=0):
    """Tensors of the given sizes; `offset` elements of misalignment in front of every one."""
    def place(a, dtype):
        t = torch.zeros(a.size + offset, dtype=dtype, device="cuda")
        t[offset:] = torch.from_numpy(a).cuda().to(dtype)
        return t[offset:]
    w = [place(rng.standard_normal(n).astype(np.float32), torch.float32) for n in sizes]
    g = [place(rng.standard_normal(n).astype(np.float32) * np.float32(10.0) ** rng.integers(-4, 1, n).astype(np.float32), DT[gdt]) for n in sizes]
    return w, g, place


def np32(t):
    return t.float().cpu().numpy()


def close(got, ref, tol):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    return got.size == 0 or np.abs(got - ref).max() <= tol * max(np.abs(ref).max(), 1e-30)


SIZES = [1, 7, 255, 256, 257, 2048, 2049, 0, 5000, 3]


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("copy", [None, "bf16", "f16"])
@pytest.mark.parametrize("gdt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dynamic", [True, False])
def test_fp32_moments(ops, gdt, copy, offset, dynamic):
    rng = np.random.default_rng(1)
    w, g, place = make(rng, SIZES, gdt, offset)
    m = [place(rng.standard_normal(n).astype(np.float32) * 0.1, torch.float32) for n in SIZES]
    v = [place(rng.random(n).astype(np.float32) * 0.1, torch.float32) for n in SIZES]
    cp = None if copy is None else [place(np.zeros(n, np.float32), DT[copy]) for n in SIZES]
    wd = [0.1 * (k % 3) for k in range(len(SIZES))]
    clip = torch.full((1,), 0.7, device="cuda")
    before = [[np32(t) for t in ts] for ts in (w, g, m, v)]
    ops.adam_multi(ops.AdamTensors(w, g, m, v, copy=cp, wd=wd), **HYPER, gscale=0.5, clip=clip, dynamic=dynamic)
    clip = float(np.float32(0.7))
    for k in range(len(SIZES)):
        w0, g0, m0, v0 = (b[k].astype(np.float64) for b in before)
        rw, rm, rv = update64(w0, g0, m0, v0, **HYPER, wd=wd[k], gscale=0.5, clip=clip, dynamic=dynamic)
        assert close(np32(w[k]), rw, 2e-6) and close(np32(m[k]), rm, 2e-6) and close(np32(v[k]), rv, 2e-6), SIZES[k]
        if cp is not None:
            assert torch.equal(cp[k], w[k].to(DT[copy]))


@pytest.mark.gpu
def test_equals_the_flat_step_bit_for_bit(ops):
    rng = np.random.default_rng(2)
    w, g, place = make(rng, [4096, 1000], "f32")
    m, v = [torch.rand_like(t) for t in w], [torch.rand_like(t) for t in w]
    other = [[t.clone() for t in ts] for ts in (w, m, v)]
    ops.adam_multi(ops.AdamTensors(w, g, m, v, wd=0.1), **HYPER, gscale=0.25)
    for k in range(2):
        ops.adam(other[0][k], g[k], other[1][k], other[2][k], HYPER["t"], HYPER["lr"], HYPER["b1"], HYPER["b2"], HYPER["eps"], wd=0.1, gscale=0.25)
        assert torch.equal(w[k], other[0][k]) and torch.equal(m[k], other[1][k]) and torch.equal(v[k], other[2][k])


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("gdt", ["f32", "bf16", "f16"])
def test_8_bit_moments(ops, gdt, offset):
    """Codes, scales and weights over several steps, each from the stored state of the one before."""
    rng = np.random.default_rng(3)
    w, g, place = make(rng, SIZES, gdt, offset)
    blocks = [-(-n // BLOCK) for n in SIZES]
    m, v = ([place(np.zeros(n, np.float32), torch.uint8) for n in SIZES] for _ in range(2))
    ms, vs = ([torch.zeros(b, device="cuda") for b in blocks] for _ in range(2))
    tensors = ops.AdamTensors(w, g, m, v, m_scale=ms, v_scale=vs, wd=0.1)
    for step in range(1, 5):
        before = [[t.cpu().numpy() if t.dtype == torch.uint8 else np32(t) for t in ts] for ts in (w, g, m, v, ms, vs)]
        h = dict(HYPER, t=step)
        ops.adam_multi(tensors, **h, seed=step)
        for k, n in enumerate(SIZES):
            w0, g0, cm, cv, sm, sv = (b[k] for b in before)
            m0, v0 = decode(cm, sm, False), decode(cv, sv, True)
            rw, _, _ = update64(w0.astype(np.float64), g0.astype(np.float64), m0.astype(np.float64), v0.astype(np.float64), **h, wd=0.1, gscale=1.0, clip=1.0, dynamic=True)
            assert close(np32(w[k]), rw, 2e-6), (step, n)
            m1, v1 = moments32(g0, m0, v0, h["b1"], h["b2"], 1.0, 1.0)
            for got, scale, value, second in ((m[k], ms[k], m1, False), (v[k], vs[k], v1, True)):
                c, s = encode(value, step, k, second)
                assert np.array_equal(got.cpu().numpy(), c) and np.array_equal(np32(scale), s), (step, n, second)
        for ts in g:                                       # other gradients, some zero
            ts.mul_(-0.3).masked_fill_(torch.rand(ts.shape, device="cuda") < 0.2, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 256, 1000, 70001])
@pytest.mark.parametrize("second", [False, True])
def test_pack_and_unpack(ops, n, second):
    rng = np.random.default_rng(4)
    x = rng.standard_normal(n).astype(np.float32) * np.float32(10.0) ** rng.integers(-6, 3, n).astype(np.float32)
    x = np.abs(x) if second else x
    codes, scales = ops.adam_state_pack(torch.from_numpy(x).cuda(), second, seed=9)
    c, s = encode(x, 9, 0, second)
    assert np.array_equal(codes.cpu().numpy(), c) and np.array_equal(np32(scales), s)
    got = np32(ops.adam_state_unpack(codes, scales, second))
    assert np.array_equal(got, decode(c, s, second))
    # a code is off by less than one spacing: 1/8 of the value, or the smallest code's value below the normal range
    tiny = np.repeat(s, BLOCK)[:n].astype(np.float64) * (2.0 ** -17 if second else 2.0 ** -9)
    assert (np.abs(got - x) <= np.maximum(np.abs(x) / 8, tiny) * (1 + 1e-6)).all()
    if second:
        assert (got[x > 0] > 0).all()


@pytest.mark.gpu
def test_zero_tiny_and_nonfinite_blocks(ops):
    x = torch.zeros(5 * BLOCK, device="cuda")
    x[BLOCK:2 * BLOCK] = 1e-35                             # below 2^-100: stored as zeros
    x[2 * BLOCK] = float("nan")
    x[2 * BLOCK + 1] = 1.0
    x[3 * BLOCK + 5] = float("inf")
    x[4 * BLOCK:] = 3.0
    for second in (False, True):
        got = ops.adam_state_unpack(*ops.adam_state_pack(x, second), second)
        assert bool((got[:2 * BLOCK] == 0).all()) and bool(got[2 * BLOCK:4 * BLOCK].isnan().all())
        # 3 is coded as 3 * inverse, within two roundings of the top code; the code below it is taken with a probability of
        # that error over the spacing, under 2^-19.  The top code then stands for top * (3 * (1 / top)): three roundings of
        # half a step, 3 * 2^-24 of the value.
        assert bool(((got[4 * BLOCK:] - 3.0).abs() <= 3.0 * 3 * 2.0 ** -24).all())


@pytest.mark.gpu
def test_many_tensors_in_several_launches(ops):
    """More tensors than one launch holds: the noise goes by the place in the whole list."""
    count = 900
    g = [torch.full((3,), 0.1 * (k + 1), device="cuda") for k in range(count)]
    w, m, v = ([torch.zeros(3, device="cuda") for _ in range(count)] for _ in range(3))
    q = [[torch.zeros(3, dtype=torch.uint8, device="cuda") for _ in range(count)] for _ in range(2)]
    s = [[torch.zeros(1, device="cuda") for _ in range(count)] for _ in range(2)]
    w8 = [t.clone() for t in w]
    ops.adam_multi(ops.AdamTensors(w, g, m, v), **HYPER)
    ops.adam_multi(ops.AdamTensors(w8, g, *q, *s), **HYPER, seed=11)
    for k in (0, 399, 400, 799, 800, 899):
        # from zero weights the step itself: root and quotient within 2^-22 each beside 8-bit states, five roundings more
        assert bool(((w[k] - w8[k]).abs() <= (2 * 2.0 ** -22 + 6 * 2.0 ** -24) * w[k].abs()).all()) and float(m[k][0]) != 0.0
        assert np.array_equal(q[1][k].cpu().numpy(), encode(np32(v[k]), 11, k, True)[0])


@pytest.mark.gpu
def test_captured_step_replays_and_empty_list(ops):
    rng = np.random.default_rng(5)
    w, g, _ = make(rng, [1000, 300], "bf16")
    m, v = [torch.zeros_like(t) for t in w], [torch.zeros_like(t) for t in w]
    twin = [[t.clone() for t in ts] for ts in (w, m, v)]
    tensors = ops.AdamTensors(w, g, m, v)
    ops.adam_multi(ops.AdamTensors([], [], [], []), **HYPER)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.adam_multi(tensors, **HYPER)
    for _ in range(3):
        graph.replay()
        ops.adam_multi(ops.AdamTensors(twin[0], g, twin[1], twin[2]), **HYPER)
    assert all(torch.equal(a, b) for x, y in zip((w, m, v), twin) for a, b in zip(x, y))


@pytest.mark.gpu
def test_refusals(ops):
    L = lib.load()
    t = [torch.zeros(8, device="cuda") for _ in range(4)]
    item = (lib.AdamItem * 1)(lib.AdamItem(8, *[a.data_ptr() for a in t], None, None, None, 0.0, 0))

    def call(state=0, g=0, cp=1, count=1, items=item, step=1, flags=1):
        return L.ane_cuda_adam_multi_dev(None, state, g, cp, count, items, step, 1e-3, 0.9, 0.9, 1e-8, 1.0, None, 0, flags)
    assert call() == lib.OK
    for bad in (dict(state=2), dict(g=3), dict(count=-1), dict(items=None), dict(step=0), dict(flags=2), dict(state=1)):
        assert call(**bad) == lib.ERR_INVALID, bad
    item[0].copy = t[0].data_ptr()
    assert call(cp=0) == lib.ERR_INVALID
    item[0].copy = None
    item[0].w = None
    assert call() == lib.ERR_INVALID
    item[0].w = t[0].data_ptr() + 2
    assert call() == lib.ERR_INVALID
    lib.set_tuning("check_extents", 1)
    try:
        item[0].w = t[2].data_ptr()                        # the same memory as m
        assert call() == lib.ERR_INVALID
        item[0].w, item[0].g = t[0].data_ptr(), t[3].data_ptr()        # the gradient in the memory of v
        assert call() == lib.ERR_INVALID
        item[0].g = t[1].data_ptr()
        assert call() == lib.OK
    finally:
        lib.clear_tuning("check_extents")
    assert L.ane_cuda_adam_state_unpack_dev(None, 8, None, None, None, 0) == lib.ERR_INVALID
    assert L.ane_cuda_adam_state_pack_dev(None, 8, t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), 2, 0) == lib.ERR_INVALID

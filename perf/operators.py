"""Timing cases of three operators of the training step: the norms around a block (``block_norm``), the loss head
without logits (``linear_cross_entropy``) and the AdamW step over a list of tensors (``adam_multi``).

``run`` computes an operator in plain torch operations, or with ``own = True`` through ``ane_b200.dev_ops``.  Both forms
update what the operator updates (accumulated gradients, weights, optimizer states) in the state's own buffers.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 256                     # elements of an 8-bit optimizer state that share a scale
EPS = 1e-5


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one fp32 sequence of the small reference model (dim 768, 256 tokens): a latency
        {"name": "block norm, one sequence", "op": "norm", "backward": False, "dtype": "float32", "B": 1, "C": 768, "S": 256,
         "gate": "channel", "post": True},
        # a micro-batch of the large configuration: 32 sequences of 2048 tokens, dim 1024
        {"name": "block norm, micro-batch", "op": "norm", "backward": False, "dtype": "bfloat16", "B": 32, "C": 1024, "S": 2048,
         "gate": "channel", "post": True},
        # its backward pass, with a gate of its own for every sequence (a conditioned block)
        {"name": "block norm bwd, micro-batch", "op": "norm", "backward": True, "dtype": "bfloat16", "B": 32, "C": 1024, "S": 2048,
         "gate": "sequence", "post": True},
        # odd channel count and odd length, no gate: rows that break every 16-byte alignment
        {"name": "block norm bwd, ragged", "op": "norm", "backward": True, "dtype": "float16", "B": 5, "C": 1000, "S": 333,
         "gate": "none", "post": True},
        # a reference training step's classifier: fp32, one sequence, the compacted vocabulary
        {"name": "loss head, one sequence", "op": "xent", "backward": True, "dtype": "float32", "B": 1, "D": 768, "V": 9200, "S": 256},
        # the large vocabulary with its gradients, 8192 tokens
        {"name": "loss head, large vocabulary", "op": "xent", "backward": True, "dtype": "bfloat16", "B": 4, "D": 1024, "V": 151936, "S": 2048},
        # evaluation of padded sequences of odd length: the loss of every token
        {"name": "loss only, odd length", "op": "xent", "backward": False, "dtype": "float16", "B": 3, "D": 768, "V": 32000, "S": 515},
        # scoring a short continuation: the table is read for a few tokens
        {"name": "loss only, few tokens", "op": "xent", "backward": False, "dtype": "bfloat16", "B": 1, "D": 1024, "V": 151936, "S": 16},
        # a toy model: all launch latency
        {"name": "adamw, toy model", "op": "adam", "bits": 32, "grads": "float32", "copy": False, "dim": 64, "hidden": 176, "layers": 2, "V": 512},
        # the small reference model (110 M parameters, 110 tensors), fp32 states
        {"name": "adamw 32-bit, 110M", "op": "adam", "bits": 32, "grads": "float32", "copy": False, "dim": 768, "hidden": 2048, "layers": 12, "V": 32000},
        # the same in mixed precision: 8-bit states, bf16 gradients, a bf16 copy of the weights for the products
        {"name": "adamw 8-bit, 110M", "op": "adam", "bits": 8, "grads": "bfloat16", "copy": True, "dim": 768, "hidden": 2048, "layers": 12, "V": 32000},
        # odd dimensions: tensors that end inside a block of 256
        {"name": "adamw 8-bit, odd sizes", "op": "adam", "bits": 8, "grads": "float32", "copy": True, "dim": 333, "hidden": 911, "layers": 6, "V": 5003},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "xent", "adam"])
    if op == "norm":
        C, S = _log_int(rng, 64, 4096), _log_int(rng, 1, 4096)
        if rng.random() < 0.5:
            C, S = -(-C // 64) * 64, -(-S // 8) * 8
        B = _log_int(rng, 1, max(1, min(64, (1 << 26) // (C * S))))
        return {"op": op, "backward": rng.random() < 0.5, "dtype": rng.choice(sorted(DTYPES)), "B": B, "C": C, "S": S,
                "gate": rng.choice(["none", "channel", "sequence"]), "post": rng.random() < 0.75}
    if op == "xent":
        D, V, S = _log_int(rng, 64, 2048), _log_int(rng, 500, 152000), _log_int(rng, 1, 2048)
        if rng.random() < 0.6:
            D = -(-D // 64) * 64
        B = _log_int(rng, 1, max(1, min(16, int(4.0e11 / (D * V * S)))))
        return {"op": op, "backward": rng.random() < 0.6, "dtype": rng.choice(sorted(DTYPES)), "B": B, "D": D, "V": V, "S": S}
    dim, layers, V = _log_int(rng, 32, 800), rng.randint(1, 12), _log_int(rng, 200, 32000)
    return {"op": op, "bits": rng.choice([8, 32]), "grads": rng.choice(sorted(DTYPES)), "copy": rng.random() < 0.5, "dim": dim,
            "hidden": int(dim * rng.uniform(2.0, 2.66)), "layers": layers, "V": V}


def _adam_sizes(case):
    """(elements, decayed) of every tensor of the model: matrices and the table are decayed, norm weights are not."""
    d, h = case["dim"], case["hidden"]
    layer = [(d * d, True)] * 4 + [(h * d, True)] * 3 + [(d, False)] * 2
    return layer * case["layers"] + [(d, False), (case["V"] * d, True)]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)

    if case["op"] == "norm":
        B, C, S, dt = case["B"], case["C"], case["S"], DTYPES[case["dtype"]]
        s = {"case": case, "alpha": 0.35, "w_pre": randn(C, scale=0.1, shift=1.0),
             "w_post": randn(C, scale=0.1, shift=1.0) if case["post"] else None, "gate": None,
             "f": randn(B, C, S, dtype=dt, scale=2.0), "x": randn(B, C, S, dtype=dt)}
        if case["gate"] != "none":
            s["gate"] = randn(*((B, C) if case["gate"] == "sequence" else (C,)), scale=0.3, shift=0.5)
        if case["backward"]:
            # x is then the stored sum x2 of the forward pass; the parameter gradients are accumulated into
            s |= {"dy": randn(B, C, S, dtype=dt), "dx2": randn(B, C, S, dtype=dt, scale=0.5), "dw_pre": randn(C),
                  "dw_post": randn(C) if case["post"] else None, "dgate": None if s["gate"] is None else randn(*s["gate"].shape)}
        return s
    if case["op"] == "xent":
        B, D, V, S, dt = case["B"], case["D"], case["V"], case["S"], DTYPES[case["dtype"]]
        targets = torch.randint(0, V, (B, S), generator=g, device="cuda", dtype=torch.int32)
        # padded tails of different lengths carry no target
        keep = S - torch.randint(0, S // 8 + 1, (B, 1), generator=g, device="cuda")
        targets[torch.arange(S, device="cuda")[None, :] >= keep] = -1
        s = {"case": case, "x": randn(B, D, S, dtype=dt), "table": randn(V, D, dtype=dt, scale=1.0 / math.sqrt(D)), "targets": targets}
        if case["backward"]:
            s["d_table"] = randn(V, D, scale=1e-4)
        return s
    sizes = _adam_sizes(case)
    starts, n = [], 0
    for size, _ in sizes:                                # every tensor begins at a multiple of the block in its flat buffer
        starts.append(n)
        n += -(-size // BLOCK) * BLOCK
    rows = n // BLOCK
    live = torch.zeros(n, device="cuda")
    for a, (size, _) in zip(starts, sizes):
        live[a:a + size] = 1.0

    def views(flat):
        return [flat[a:a + size] for a, (size, _) in zip(starts, sizes)]

    def block_views(flat):
        return [flat[a // BLOCK:a // BLOCK + -(-size // BLOCK)] for a, (size, _) in zip(starts, sizes)]

    w = randn(n, scale=0.02) * live
    # gradients of a trained model: their sizes differ by orders of magnitude from row to row
    spread = torch.exp(randn(rows, scale=2.0)).repeat_interleave(BLOCK)
    s = {"case": case, "n": n, "w": w, "g": (randn(n, scale=1e-3) * spread * live).to(DTYPES[case["grads"]]), "t": 100, "lr": 3e-4, "b1": 0.9, "b2": 0.95,
         "eps": 1e-8, "gscale": 0.5, "clip": torch.full((1,), 0.8, device="cuda"), "seed": 1234 + seed % 1000,
         "wd": [0.1 if decayed else 0.0 for _, decayed in sizes], "sizes": [size for size, _ in sizes],
         "padded": [-(-size // BLOCK) * BLOCK for size, _ in sizes]}
    s["copy"] = torch.zeros(n, device="cuda", dtype=torch.bfloat16) if case["copy"] else None
    if case["bits"] == 32:
        s["m"], s["v"] = randn(n, scale=3e-4) * spread * live, randn(n, scale=1e-3).square() * spread.square() * live
        s["m_scale"] = s["v_scale"] = None
    else:
        # codes of an 8-bit state in use: a magnitude code for every element, a scale for every 256
        s["m"] = torch.randint(0, 256, (n,), generator=g, device="cuda").to(torch.uint8) * live.to(torch.uint8)
        s["v"] = torch.randint(64, 256, (n,), generator=g, device="cuda").to(torch.uint8) * live.to(torch.uint8)
        s["m_scale"] = torch.exp(randn(rows, scale=2.0)) * 1e-6
        s["v_scale"] = torch.exp(randn(rows, scale=2.0)) * 1e-11
    for key in ("w", "g", "copy"):
        s[key + "_list"] = None if s[key] is None else views(s[key])
    s["m_list"], s["v_list"] = views(s["m"]), views(s["v"])
    s["m_scale_list"] = None if s["m_scale"] is None else block_views(s["m_scale"])
    s["v_scale_list"] = None if s["v_scale"] is None else block_views(s["v_scale"])
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        from ane_b200 import dev_ops, lib
        lib.init(torch.cuda.current_device())
        return {"norm": _own_norm, "xent": _own_xent, "adam": _own_adam}[state["case"]["op"]](dev_ops, state)
    return {"norm": _plain_norm, "xent": _plain_xent, "adam": _plain_adam}[state["case"]["op"]](state)


def _own_norm(ops, s):
    if not s["case"]["backward"]:
        return ops.block_norm(s["x"], s["f"], s["w_pre"], w_post=s["w_post"], gate=s["gate"], alpha=s["alpha"], eps=EPS)
    dx, df = ops.block_norm_bwd(s["dy"], s["x"], s["f"], s["w_pre"], s["dw_pre"], w_post=s["w_post"], dw_post=s["dw_post"],
                                gate=s["gate"], dgate=s["dgate"], dx2=s["dx2"], alpha=s["alpha"], eps=EPS)
    return [t for t in (dx, df, s["dw_pre"], s["dw_post"], s["dgate"]) if t is not None]


def _own_xent(ops, s):
    if not s["case"]["backward"]:
        loss_tok = torch.empty_like(s["targets"], dtype=torch.float32)
        return ops.linear_cross_entropy(s["x"], s["table"], s["targets"], grad=False, loss_tok=loss_tok)[0], loss_tok
    loss, dx = ops.linear_cross_entropy(s["x"], s["table"], s["targets"], d_table=s["d_table"])
    return loss, dx, s["d_table"]


def _own_adam(ops, s):
    if "tensors" not in s:       # the list of tensors is made once, as an optimizer does
        s["tensors"] = ops.AdamTensors(s["w_list"], s["g_list"], s["m_list"], s["v_list"], m_scale=s["m_scale_list"],
                                       v_scale=s["v_scale_list"], copy=s["copy_list"], wd=s["wd"])
    ops.adam_multi(s["tensors"], s["t"], s["lr"], s["b1"], s["b2"], s["eps"], gscale=s["gscale"], clip=s["clip"], seed=s["seed"])
    m, v = s["m"], s["v"]
    if s["case"]["bits"] == 8:
        m, v = ops.adam_state_unpack(m, s["m_scale"]), ops.adam_state_unpack(v, s["v_scale"], second=True)
    return [t for t in (s["w"], m, v, s["copy"]) if t is not None]


# ------------------------------------------------------------------ the plain forms
def _channels(t):
    """[C] or [B, C] beside [B, C, S]."""
    return t[..., None] if t.dim() == 2 else t[None, :, None]


def _plain_norm(s):
    dt, alpha, f = s["x"].dtype, s["alpha"], s["f"].float()
    w_pre = _channels(s["w_pre"])
    w_post = 1.0 if s["w_post"] is None else _channels(s["w_post"])
    gate = 1.0 if s["gate"] is None else _channels(s["gate"])
    # without a norm after the block the branch is taken as it is
    rf = 1.0 if s["w_post"] is None else torch.rsqrt(f.square().mean(1, keepdim=True) + EPS)
    if not s["case"]["backward"]:
        x2 = s["x"].float() + alpha * gate * (f * rf * w_post)
        x2 = x2.to(dt)                                   # the sum is stored, and normalised as it is stored
        x2f = x2.float()
        return x2, (x2f * torch.rsqrt(x2f.square().mean(1, keepdim=True) + EPS) * w_pre).to(dt)
    x2, dy = s["x"].float(), s["dy"].float()
    r2 = torch.rsqrt(x2.square().mean(1, keepdim=True) + EPS)
    wdy = w_pre * dy
    G = s["dx2"].float() + r2 * wdy - x2 * (r2 * r2 * r2 * (wdy * x2).mean(1, keepdim=True))
    s["dw_pre"] += (dy * x2 * r2).sum((0, 2))
    fr = f * rf
    if s["gate"] is not None:
        dgate = alpha * (G * fr * w_post).sum(2)
        s["dgate"] += dgate if s["gate"].dim() == 2 else dgate.sum(0)
    dn = alpha * gate * G
    if s["w_post"] is None:
        df = dn
    else:
        s["dw_post"] += (dn * fr).sum((0, 2))
        q = w_post * dn
        df = rf * (q - fr * (q * fr).mean(1, keepdim=True))
    return [t for t in (G.to(dt), df.to(dt), s["dw_pre"], s["dw_post"], s["dgate"]) if t is not None]


def _plain_xent(s):
    B, D, S = s["x"].shape
    x, E = s["x"].float().transpose(1, 2).reshape(B * S, D), s["table"].float()
    target = s["targets"].reshape(-1).long()
    valid = (target >= 0) & (target < E.shape[0])
    at = torch.where(valid, target, 0)[:, None]
    logits = x @ E.t()
    top = logits.max(1, keepdim=True).values
    p = torch.exp(logits - top)
    p = p / p.sum(1, keepdim=True)
    loss_tok = -(torch.log(p.gather(1, at)[:, 0] + 1e-10) * valid).reshape(B, S)
    loss = loss_tok.sum(1) / S
    if not s["case"]["backward"]:
        return loss, loss_tok
    p = p.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32)) * (valid / S)[:, None]
    s["d_table"] += p.t() @ x
    return loss, (p @ E).reshape(B, S, D).transpose(1, 2).contiguous().to(s["x"].dtype), s["d_table"]


def _mix(h):
    """The finaliser of MurmurHash3 on 32-bit values held in int64."""
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def _noise(s):
    """20 random bits for each element's first and second moment, from the step's seed, the tensor's place in the list and
    the element's place in its tensor."""
    device = s["w"].device
    padded = torch.tensor(s["padded"], device=device)
    start = torch.cumsum(padded, 0) - padded
    key = _mix((s["seed"] + 0x9E3779B9 * torch.arange(len(s["padded"]), device=device)) & 0xFFFFFFFF)
    place = torch.arange(s["n"], device=device) - start.repeat_interleave(padded, output_size=s["n"])
    h = _mix((place * 0x9E3779B1 + key.repeat_interleave(padded, output_size=s["n"])) & 0xFFFFFFFF)
    return h >> 12, h & 0xFFFFF


def _decode(code, scale, second):
    """Codes stand for floats without infinities: 4 exponent and 3 mantissa bits beside a sign for the first moment
    (bias 7), 5 exponent and 3 mantissa bits for the second (bias 15), times the scale of their block of 256."""
    code = code.to(torch.int32)
    value = ((code if second else code & 127) << 20).view(torch.float32) * (2.0 ** 112 if second else 2.0 ** 120)
    value = value if second else torch.where(code >= 128, -value, value)
    return (value.view(-1, BLOCK) * scale[:, None]).view(-1)


def _encode(value, noise, second):
    """Codes and scales of fp32 values: the block's largest magnitude takes the top code, the others are rounded up or down
    with the probability that keeps their mean; a second moment above zero keeps a code above zero."""
    top = 122880.0 if second else 480.0
    most = value.abs().view(-1, BLOCK).amax(1)
    most = torch.where(most < 2.0 ** -100, torch.zeros_like(most), most)
    scale, inverse = most / top, torch.where(most > 0, top / most, torch.zeros_like(most))
    y = (value.abs().view(-1, BLOCK) * inverse[:, None]).view(-1) * (2.0 ** -112 if second else 2.0 ** -120)
    code = (y.view(torch.int32).to(torch.int64) + noise >> 20).clamp(max=255 if second else 127)
    code = torch.where((code == 0) & (y > 0), 1, code) if second else torch.where(value < 0, code + 128, code)
    return code.to(torch.uint8), scale


def _plain_adam(s):
    one, b1, b2 = np.float32(1), np.float32(s["b1"]), np.float32(s["b2"])
    quantised = s["case"]["bits"] == 8
    g = s["g"].float() * s["gscale"] * s["clip"]
    m = _decode(s["m"], s["m_scale"], False) if quantised else s["m"]
    v = _decode(s["v"], s["v_scale"], True) if quantised else s["v"]
    m = m * float(b1) + g * float(one - b1)
    v = v * float(b2) + g * float(one - b2) * g
    mh, vh = m / (1 - s["b1"] ** s["t"]), v / (1 - s["b2"] ** s["t"])
    device = s["w"].device
    wd = torch.tensor(s["wd"], device=device).repeat_interleave(torch.tensor(s["padded"], device=device), output_size=s["n"])
    s["w"] -= s["lr"] * (mh / (vh.sqrt() + s["eps"]) + wd * s["w"])
    if s["copy"] is not None:
        s["copy"].copy_(s["w"])
    if not quantised:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return [t for t in (s["w"], s["m"], s["v"], s["copy"]) if t is not None]
    noise_m, noise_v = _noise(s)
    for_m, for_v = _encode(m, noise_m, False), _encode(v, noise_v, True)
    s["m"].copy_(for_m[0]), s["m_scale"].copy_(for_m[1])
    s["v"].copy_(for_v[0]), s["v_scale"].copy_(for_v[1])
    return [t for t in (s["w"], _decode(s["m"], s["m_scale"], False), _decode(s["v"], s["v_scale"], True), s["copy"]) if t is not None]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "norm":
        n = case["B"] * case["C"] * case["S"]
        e = 4 if case["dtype"] == "float32" else 2
        return {"bytes": (6 if case["backward"] else 4) * n * e, "flops": (40 if case["backward"] else 15) * n}
    if case["op"] == "xent":
        T, D, V = case["B"] * case["S"], case["D"], case["V"]
        e = 4 if case["dtype"] == "float32" else 2
        read = (T * D + V * D) * e + 4 * T
        return {"bytes": read + (T * D * e + 8 * V * D if case["backward"] else 4 * T), "flops": (6 if case["backward"] else 2) * T * D * V}
    n = sum(size for size, _ in _adam_sizes(case))
    per = 8 + (4 if case["grads"] == "float32" else 2) + (16 if case["bits"] == 32 else 4 + 8 + 16 / BLOCK) + (2 if case["copy"] else 0)
    return {"bytes": int(per * n), "flops": 20 * n}


# ------------------------------------------------------------------ in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "xent": _exact_xent, "adam": _exact_adam}[case["op"]](s)


def _exact_norm(s):
    case, alpha = s["case"], s["alpha"]
    B, C, S = s["x"].shape
    gate = torch.ones(B, C, dtype=torch.float64, device="cuda")
    if s["gate"] is not None:
        gate = gate * s["gate"].double()                 # [C] and [B, C] alike
    w_pre = s["w_pre"].double().view(1, C, 1)
    post = s["w_post"] is not None
    w_post = s["w_post"].double().view(1, C, 1) if post else torch.ones(1, C, 1, dtype=torch.float64, device="cuda")
    outs, grads = [], {"dw_pre": 0.0, "dw_post": 0.0, "dgate": []}
    for b in range(B):                                   # a sequence at a time keeps the 64-bit temporaries small
        f, k = s["f"][b:b + 1].double(), alpha * gate[b].view(1, C, 1)
        sigma = torch.sqrt((f * f).sum(1, keepdim=True) / C + EPS) if post else torch.ones(1, 1, S, dtype=torch.float64, device="cuda")
        unit = f / sigma
        if not case["backward"]:
            x2 = s["x"][b:b + 1].double() + k * w_post * unit
            z = x2.to(s["x"].dtype).double()
            outs.append((x2, z / torch.sqrt((z * z).sum(1, keepdim=True) / C + EPS) * w_pre))
            continue
        x2, dy = s["x"][b:b + 1].double(), s["dy"][b:b + 1].double()
        rho = torch.sqrt((x2 * x2).sum(1, keepdim=True) / C + EPS)
        z = x2 / rho
        a = w_pre * dy
        G = s["dx2"][b:b + 1].double() + (a - z * ((a * z).sum(1, keepdim=True) / C)) / rho
        grads["dw_pre"] += (dy * z).sum((0, 2))
        grads["dgate"].append((alpha * w_post * unit * G).sum(2))
        df = k * G
        if post:
            grads["dw_post"] += (df * unit).sum((0, 2))
            df = w_post * df
            df = (df - unit * ((df * unit).sum(1, keepdim=True) / C)) / sigma
        outs.append((G, df))
    outs = [torch.cat(parts) for parts in zip(*outs)]
    if not case["backward"]:
        return tuple(outs)
    outs.append(s["dw_pre"].double() + grads["dw_pre"])
    if post:
        outs.append(s["dw_post"].double() + grads["dw_post"])
    if s["gate"] is not None:
        d = torch.cat(grads["dgate"])
        outs.append(s["dgate"].double() + (d if s["gate"].dim() == 2 else d.sum(0)))
    return outs


def _exact_xent(s):
    (B, D, S), V = s["x"].shape, s["table"].shape[0]
    X = s["x"].double().permute(1, 0, 2).reshape(D, B * S)
    y = s["targets"].reshape(-1).long()
    ok = (y >= 0) & (y < V)
    piece = 8192
    Z, hit = torch.full((B * S,), -math.inf, dtype=torch.float64, device="cuda"), torch.zeros(B * S, dtype=torch.float64, device="cuda")
    for lo in range(0, V, piece):
        L = s["table"][lo:lo + piece].double() @ X
        Z = torch.logaddexp(Z, torch.logsumexp(L, 0))
        here = ok & (y >= lo) & (y < lo + L.shape[0])
        cols = here.nonzero()[:, 0]
        hit[cols] = L[y[cols] - lo, cols]
    per_token = torch.where(ok, -torch.log(torch.exp(hit - Z) + 1e-10), torch.zeros_like(hit))
    loss = per_token.view(B, S).sum(1) / S
    if not s["case"]["backward"]:
        return loss, per_token.view(B, S)
    dX, dE = torch.zeros_like(X), s["d_table"].double()
    for lo in range(0, V, piece):
        E = s["table"][lo:lo + piece].double()
        P = torch.exp(E @ X - Z)
        cols = (ok & (y >= lo) & (y < lo + E.shape[0])).nonzero()[:, 0]
        P[y[cols] - lo, cols] -= 1.0
        P *= ok / S
        dX += E.t() @ P
        dE[lo:lo + piece] += P @ X.t()
    return loss, dX.view(D, B, S).permute(1, 0, 2).contiguous(), dE


def _exact_adam(s):
    quantised = s["case"]["bits"] == 8

    def value(code, scale, exponent_bits, mantissa_bits, bias):
        """A code's value by its fields: (1 + mantissa/8) * 2^(exponent - bias), or mantissa/8 * 2^(1 - bias) below."""
        c = code.to(torch.int64)
        e, f = (c >> mantissa_bits) & ((1 << exponent_bits) - 1), (c & ((1 << mantissa_bits) - 1)).double() / (1 << mantissa_bits)
        return torch.where(e > 0, (1 + f) * torch.exp2((e - bias).double()), f * 2.0 ** (1 - bias)) * scale.double().repeat_interleave(BLOCK)

    b1, b2 = float(np.float32(s["b1"])), float(np.float32(s["b2"]))
    g = s["g"].double() * s["gscale"] * s["clip"].double()
    if quantised:
        m = value(s["m"] & 127, s["m_scale"], 4, 3, 7) * (1 - 2 * (s["m"] >> 7).double())
        v = value(s["v"], s["v_scale"], 5, 3, 15)
    else:
        m, v = s["m"].double(), s["v"].double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    decay = torch.cat([torch.full((n,), wd, dtype=torch.float64, device="cuda") for n, wd in zip(s["padded"], s["wd"])])
    w = s["w"].double()
    w = w - s["lr"] * (m / (1 - s["b1"] ** s["t"]) / (torch.sqrt(v / (1 - s["b2"] ** s["t"])) + s["eps"]) + decay * w)
    # what an 8-bit state holds afterwards hangs on where the random rounding of fp32 values falls: no 64-bit value
    outs = [w, None, None] if quantised else [w, m, v]
    return outs + ([w.clone()] if s["copy"] is not None else [])

"""Timed operators around and inside the MoE block: 4-bit microscaled experts and the fused residual norm.

  round     quantize_mx4 and its values: activations and weights to 4 bits in blocks of 32 with a shared
            power-of-two scale, and back
  product   grouped products of two such operands: mx4_grouped_mm (rows of group g times W[g]^T) and
            mx4_swiglu (the gate | up projection with silu(gate) * up)
  experts   mx4_experts: a layer's routed experts on 4-bit weights, from the hidden states to their sum
  norm      residual_norm: hidden = residual_scale * residual + branch_scale * gate * N(y; post_weight) and
            x = N(hidden; weight), forward alone (decoding) or with its gradients (training)

A microscaled row of K values is K/2 bytes (the element of even index in the low four bits; sign, two exponent
bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one byte s per 32 values, 2^(s - 127), s = 255 standing
for NaN; scales are stored in rows of 8 ceil(K/256) bytes, of which the first K/32 count.
"""

from __future__ import annotations

import math

import torch

own = False  # False: the plain forms below; True: the framework's operators

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# (hidden, experts, top_k, intermediate): the benchmark's two layers and three generic smaller ones
LAYER_30B = dict(hidden=2048, experts=128, top_k=8, inter=768)
LAYER_235B = dict(hidden=4096, experts=128, top_k=8, inter=1536)
LAYER_MID = dict(hidden=1536, experts=64, top_k=6, inter=640)
LAYER_SMALL = dict(hidden=1024, experts=32, top_k=4, inter=512)
LAYER_TINY = dict(hidden=256, experts=8, top_k=2, inter=128)
LISTED_MAX_ELEMENTS = 128 * 1536 * 2048
LISTED_MAX_FLOPS = 2.0 * 131072 * 2304 * 2048
LISTED_MAX_NORM = 16384 * 2048


def listed() -> list[dict]:
    return [
        # the activations of a decoding batch on their way into the experts: latency
        dict(name="round_48", op="round", sheets=1, rows=48, k=2048, dtype="bf16"),
        # a layer's gate and up weights, quantised once at load time
        dict(name="round_weights", op="round", sheets=128, rows=1536, k=2048, dtype="bf16"),
        # the gate and up projection of 48 decoding tokens: a few rows for most experts, the weights stream once
        dict(name="swiglu_384", op="product", swiglu=True, rows=384, groups=128, n=768, k=2048, skew=0.0),
        # the same projection in the prefill of a 1531-token prompt
        dict(name="swiglu_12248", op="product", swiglu=True, rows=12248, groups=128, n=768, k=2048, skew=0.0),
        # the down projection on an expert-parallel rank's rows: 64 local experts, Zipf routing, some without rows
        dict(name="down_10007_zipf", op="product", swiglu=False, rows=10007, groups=64, n=2048, k=768, skew=1.2),
        # the wide layer's down projection over 8192 tokens
        dict(name="down_65536", op="product", swiglu=False, rows=65536, groups=128, n=4096, k=1536, skew=0.0),
        # one token through a layer's experts: latency and launches
        dict(name="experts_1", op="experts", tokens=1, **LAYER_30B),
        # a long prefill (or a batch of them): 16384 tokens
        dict(name="experts_16384", op="experts", tokens=16384, **LAYER_30B),
        # one decoding token between two blocks: the residual sum and the next norm, no gradients
        dict(name="norm_1", op="norm", rows=1, h=2048, dtype="bf16", post=False, gate="none", scaled=False, train=False),
        # the same in a training step of 16384 tokens
        dict(name="norm_16384_train", op="norm", rows=16384, h=2048, dtype="bf16", post=False, gate="none", scaled=False,
             train=True),
        # norms on both sides of the block, its output gated per token and scaled, a padded batch of odd length
        dict(name="norm_5003_sandwich_train", op="norm", rows=5003, h=4096, dtype="bf16", post=True, gate="token",
             scaled=True, train=True),
        # full precision with a learned gate per channel
        dict(name="norm_2047_fp32_train", op="norm", rows=2047, h=1536, dtype="fp32", post=True, gate="channel",
             scaled=True, train=True),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """A whole number spread evenly over the logarithm of its range."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["round", "product", "product", "product", "experts", "experts", "norm", "norm", "norm"])
    if op == "round":
        k = 32 * _log(rng, 1, 256)
        rows = _log(rng, 1, max(1, min(1 << 18, LISTED_MAX_ELEMENTS // (2 * k))))
        sheets = 1 if rng.random() < 0.7 else rng.randint(2, 9)
        return dict(op=op, sheets=sheets, rows=max(1, rows // sheets), k=k, dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if op == "product":
        swiglu = rng.random() < 0.5
        if rng.random() < 0.5:
            layer = rng.choice([LAYER_30B, LAYER_235B, LAYER_MID, LAYER_SMALL])
            groups = layer["experts"]
            n, k = (layer["inter"], layer["hidden"]) if swiglu else (layer["hidden"], layer["inter"])
        else:
            groups, n, k = rng.choice([1, 2, 5, 16, 33, 64, 160]), 8 * _log(rng, 1, 320), 32 * _log(rng, 1, 80)
        most = int(LISTED_MAX_FLOPS / (2.0 * k * n * (2 if swiglu else 1)))
        return dict(op=op, swiglu=swiglu, rows=_log(rng, 1, max(1, min(65536, most))), groups=groups, n=n, k=k,
                    skew=rng.choice([0.0, 0.0, 0.8, 1.2]))
    if op == "experts":
        layer = rng.choice([LAYER_30B, LAYER_30B, LAYER_235B, LAYER_MID, LAYER_SMALL, LAYER_TINY])
        return dict(op=op, tokens=_log(rng, 1, 4096 if layer is LAYER_235B else 12000), **layer)
    h = 8 * _log(rng, 1, 1024)
    return dict(op=op, rows=_log(rng, 1, max(1, min(32768, LISTED_MAX_NORM // (2 * h)))), h=h,
                dtype=rng.choice(["bf16", "bf16", "fp32"]), post=rng.random() < 0.5,
                gate=rng.choice(["none", "token", "channel", "full"]), scaled=rng.random() < 0.5,
                train=rng.random() < 0.7)


# ------------------------------------------------------------------- inputs


class _Rand:
    """Seeded normal tensors on the GPU."""

    def __init__(self, seed: int):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=self.gen, device="cuda", dtype=dtype).mul_(std)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device="cuda", dtype=torch.float32)


def _activations(r: _Rand, rows: int, k: int) -> torch.Tensor:
    """Rows of differing size with a few large channels, as normalised hidden states have them."""
    x = r.normal(rows, k)
    return x.mul_(torch.exp(r.normal(rows, 1, std=0.5))).mul_(torch.exp(r.normal(1, k, std=0.7)))


def _packed(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """What a program that holds 4-bit data keeps of x: (codes [..., K/2], scales [..., 8 ceil(K/256)]), made in slices."""
    k = x.shape[-1]
    flat = x.reshape(-1, k)
    codes = torch.empty(flat.shape[0], k // 2, dtype=torch.uint8, device=x.device)
    scales = torch.zeros(flat.shape[0], 8 * -(-k // 256), dtype=torch.uint8, device=x.device)
    step = max(1, (1 << 26) // k)
    for i in range(0, flat.shape[0], step):
        level, exponent = _levels(flat[i:i + step].float())
        level = level.reshape(-1, k)
        code = _LEVEL_CODES.to(x.device)[(2 * level.abs()).to(torch.int64)] | (8 * torch.signbit(level)).to(torch.uint8)
        codes[i:i + step] = code[:, 0::2] | (code[:, 1::2] << 4)
        scales[i:i + step, :k // 32] = (exponent.reshape(-1, k // 32) + 127).to(torch.uint8)
    return codes.reshape(*x.shape[:-1], -1), scales.reshape(*x.shape[:-1], -1)


_LEVEL_CODES = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], dtype=torch.uint8)  # code of the level index/2
_CODE_LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0])


def _counts(r: _Rand, rows: int, groups: int, skew: float) -> list[int]:
    """Rows per group: a draw with weights rank^-skew over shuffled groups."""
    weight = (torch.argsort(r.uniform(groups)) + 1.0).pow(-skew)
    picks = torch.multinomial(weight, rows, replacement=True, generator=r.gen)
    return torch.bincount(picks, minlength=groups).tolist()


def prepare(case: dict, seed: int) -> dict:
    r = _Rand(seed)
    op = case["op"]
    if op == "round":
        k, rows = case["k"], case["sheets"] * case["rows"]
        x = r.normal(rows, k, dtype=DTYPES[case["dtype"]])
        x.mul_(torch.exp(r.normal(rows, 1, std=2.0)).to(x.dtype)).mul_(0.05)
        x[torch.randint(rows, (1 + rows // 64,), generator=r.gen, device="cuda"), :32] = 0.0  # blocks of zeros
        return dict(op=op, x=x.reshape(case["sheets"], case["rows"], k).squeeze(0))
    if op == "product":
        rows, g, n, k = case["rows"], case["groups"], case["n"], case["k"]
        counts = _counts(r, rows, g, case["skew"])
        offsets = torch.tensor(counts, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
        a = _packed(_activations(r, rows, k).to(torch.bfloat16))
        w = _packed(r.normal(g, (2 if case["swiglu"] else 1) * n, k, std=0.02, dtype=torch.bfloat16))
        return dict(op=op, swiglu=case["swiglu"], a=a, w=w, offsets=offsets, counts=counts)
    if op == "experts":
        t, h, e, k, i = (case[s] for s in ("tokens", "hidden", "experts", "top_k", "inter"))
        x = _activations(r, t, h).to(torch.bfloat16)
        top = torch.topk(r.normal(t, e), k, dim=1)
        gate_up = _packed(r.normal(e, 2 * i, h, std=0.02, dtype=torch.bfloat16))
        down = _packed(r.normal(e, h, i, std=0.02, dtype=torch.bfloat16))
        counts = torch.bincount(top.indices.reshape(-1), minlength=e).tolist()
        return dict(op=op, x=x, idx=top.indices, weights=torch.softmax(top.values, dim=1), gate_up=gate_up, down=down,
                    counts=counts)
    t, h, dt = case["rows"], case["h"], DTYPES[case["dtype"]]
    shape = {"none": None, "token": (t, 1), "channel": (h,), "full": (t, h)}[case["gate"]]
    leaf = lambda x: x.to(dt).requires_grad_(case["train"])  # noqa: E731
    state = dict(op=op, train=case["train"], eps=1e-6, branch_scale=0.22 if case["scaled"] else 1.0,
                 residual_scale=1.5 if case["scaled"] else 1.0,
                 y=leaf(r.normal(t, h, std=0.7)), residual=leaf(r.normal(t, h, std=2.0)),
                 weight=leaf(1.0 + r.normal(h, std=0.2)),
                 post_weight=leaf(1.0 + r.normal(h, std=0.2)) if case["post"] else None,
                 gate=leaf(torch.sigmoid(r.normal(*shape))) if shape else None)
    state["d_hidden"], state["d_x"] = r.normal(t, h).to(dt), r.normal(t, h).to(dt)
    return state


# -------------------------------------------------------------- plain forms


def _levels(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] in blocks of 32: (levels [..., K/32, 32], the blocks' exponents), x being near level * 2^exponent:
    2^exponent is a quarter of the largest power of two in the block's largest size, and a level the nearest of 0, 0.5,
    1, 1.5, 2, 3, 4, 6 (halfway: the even one)."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    exponent = (torch.frexp(top).exponent - 3).clamp(min=-127)
    exponent = torch.where(top > 0, exponent, torch.full_like(exponent, -127))
    v = torch.ldexp(b, -exponent).clamp(-6.0, 6.0)
    size = v.abs()
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0)).to(x.dtype)
    return torch.round(v / step) * step, exponent


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The values (fp32) of codes [..., K/2] and scales [..., 8 ceil(K/256)]."""
    v = _CODE_LEVELS.to(codes.device)[torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).to(torch.int32)]
    s = torch.exp2(scales[..., :v.shape[-1] // 32].float() - 127.0)
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _rounded(x: torch.Tensor) -> torch.Tensor:
    level, exponent = _levels(x)
    return torch.ldexp(level, exponent).flatten(-2)


def _swiglu(gate_up: torch.Tensor) -> torch.Tensor:
    gate, up = gate_up.chunk(2, dim=-1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _spans(counts: list[int]) -> list[tuple[int, int, int]]:
    """(group, first row, row behind the last) of the groups that have rows."""
    ends = torch.tensor(counts).cumsum(0).tolist()
    return [(g, end - n, end) for g, (n, end) in enumerate(zip(counts, ends)) if n]


def _round_plain(s):
    return _rounded(s["x"].float()).to(s["x"].dtype)


def _product_plain(s):
    a = _values(*s["a"])
    parts = []
    for g, lo, hi in _spans(s["counts"]):
        c = a[lo:hi] @ _values(s["w"][0][g], s["w"][1][g]).t()
        parts.append((_swiglu(c) if s["swiglu"] else c).to(torch.bfloat16))
    return torch.cat(parts)


def _experts_plain(s):
    x = _rounded(s["x"].float())
    order = torch.argsort(s["idx"].reshape(-1), stable=True)
    token = order // s["idx"].shape[1]
    weight = s["weights"].float().reshape(-1)[order].unsqueeze(1)
    out = torch.zeros_like(x)
    for e, lo, hi in _spans(s["counts"]):
        act = _swiglu(x[token[lo:hi]] @ _values(s["gate_up"][0][e], s["gate_up"][1][e]).t())
        y = _rounded(act) @ _values(s["down"][0][e], s["down"][1][e]).t()
        out.index_add_(0, token[lo:hi], y * weight[lo:hi])
    return out.to(torch.bfloat16)


def _norm_plain(y, residual, weight, post_weight, gate, branch_scale, residual_scale, eps):
    dt = y.dtype
    y, residual, weight = y.float(), residual.float(), weight.float()
    if post_weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * post_weight.float()
    if gate is not None:
        y = y * gate.float()
    hidden = residual_scale * residual + branch_scale * y
    x = hidden * torch.rsqrt(hidden.square().mean(-1, keepdim=True) + eps) * weight
    return hidden.to(dt), x.to(dt)


def _leaves(s) -> dict:
    return {n: s[n] for n in ("y", "residual", "weight", "post_weight", "gate") if s[n] is not None}


def _norm_run(s, norm):
    with torch.set_grad_enabled(s["train"]):
        hidden, x = norm(s["y"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"],
                         branch_scale=s["branch_scale"], residual_scale=s["residual_scale"], eps=s["eps"])
    if not s["train"]:
        return {"hidden": hidden, "x": x}
    leaves = _leaves(s)
    grads = torch.autograd.grad([hidden, x], list(leaves.values()), [s["d_hidden"], s["d_x"]])
    return {"hidden": hidden.detach(), "x": x.detach(), **{"d_" + n: g for n, g in zip(leaves, grads)}}


def run(state: dict):
    op = state["op"]
    if own:
        import parallel_amd as pa

        if op == "round":
            return pa.quantize_mx4(state["x"]).dequantize(state["x"].dtype)
        if op == "product":
            product = pa.mx4_swiglu if state["swiglu"] else pa.mx4_grouped_mm
            return product(pa.MX4Tensor(*state["a"]), pa.MX4Tensor(*state["w"]), state["offsets"])
        if op == "experts":
            return pa.mx4_experts(state["x"], state["idx"], state["weights"], pa.MX4Tensor(*state["gate_up"]),
                                  pa.MX4Tensor(*state["down"]))
        return _norm_run(state, pa.residual_norm)
    if op == "round":
        return _round_plain(state)
    if op == "product":
        return _product_plain(state)
    if op == "experts":
        return _experts_plain(state)
    return _norm_run(state, _norm_plain)


# ------------------------------------------------------------- work and exact


def _mx_bytes(values: float) -> float:
    return values * (0.5 + 1.0 / 32.0)


def work(case: dict) -> dict:
    op = case["op"]
    if op == "round":
        n = case["sheets"] * case["rows"] * case["k"]
        return {"bytes": 2 * n * DTYPES[case["dtype"]].itemsize, "flops": 2 * n}
    if op == "product":
        rows, g, n, k = case["rows"], case["groups"], case["n"], case["k"]
        wide = n * (2 if case["swiglu"] else 1)
        hit = g * (1.0 - (1.0 - 1.0 / g) ** rows)
        return {"bytes": int(_mx_bytes(rows * k) + _mx_bytes(hit * wide * k) + 2 * rows * n + 4 * g),
                "flops": 2 * rows * wide * k}
    if op == "experts":
        t, h, e, k, i = (case[s] for s in ("tokens", "hidden", "experts", "top_k", "inter"))
        hit = e * (1.0 - (1.0 - k / e) ** t)
        return {"bytes": int(4 * t * h + 12 * t * k + _mx_bytes(hit * 3 * i * h)), "flops": 6 * t * k * h * i}
    t, h, size = case["rows"], case["h"], DTYPES[case["dtype"]].itemsize
    vectors = {"none": 0, "token": t, "channel": h, "full": t * h}[case["gate"]] + h * (2 if case["post"] else 1)
    # forward: y, residual in, hidden, x out; the gradients: d_hidden, d_x in, d_y, d_residual out (y and residual once)
    return {"bytes": size * ((8 if case["train"] else 4) * t * h + (2 if case["train"] else 1) * vectors),
            "flops": (40 if case["train"] else 12) * t * h}


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_block_values(x: torch.Tensor) -> torch.Tensor:
    """Each block of 32 on its grid, in float64: nearest grid value by comparison with the midpoints."""
    shape = x.shape
    x = x.double().reshape(-1, 32)
    top = x.abs().max(dim=1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    e = torch.where(torch.exp2(e) > top, e - 1, torch.where(torch.exp2(e + 1) <= top, e + 1, e))
    scale = torch.exp2(torch.where(top > 0, (e - 2).clamp(min=-127.0), torch.full_like(e, -127.0)))
    ratio = x.abs() / scale
    got = torch.zeros_like(ratio)
    for n in range(7):  # halfway goes to the value of even code
        middle = 0.5 * (_E2M1[n] + _E2M1[n + 1])
        got = torch.where(ratio > middle if n % 2 == 0 else ratio >= middle, torch.full_like(got, _E2M1[n + 1]), got)
    return (torch.copysign(got, x) * scale).reshape(shape)


def _exact_unpack(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    k = 2 * codes.shape[-1]
    out = torch.empty(*codes.shape[:-1], k, dtype=torch.float64, device=codes.device)
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=codes.device)
    for half in range(2):
        c = (codes >> (4 * half)) & 15
        out[..., half::2] = grid[(c & 7).long()] * (1.0 - 2.0 * (c >> 3).double())
    factor = torch.pow(2.0, scales[..., :k // 32].double() - 127.0)
    return out * factor.repeat_interleave(32, dim=-1)


def _exact_act(pre: torch.Tensor) -> torch.Tensor:
    half = pre.shape[-1] // 2
    return pre[..., :half] * torch.special.expit(pre[..., :half]) * pre[..., half:]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    op = case["op"]
    if op == "round":
        x = s["x"]
        out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        flat, into = x.reshape(-1, case["k"]), out.reshape(-1, case["k"])
        step = max(1, (1 << 25) // case["k"])
        for i in range(0, flat.shape[0], step):
            into[i:i + step] = _exact_block_values(flat[i:i + step])
        return out
    if op == "product":
        out = torch.empty(case["rows"], case["n"], dtype=torch.float64, device="cuda")
        lo = 0
        for g, count in enumerate(s["counts"]):
            if count:
                rows = _exact_unpack(s["a"][0][lo:lo + count], s["a"][1][lo:lo + count])
                c = torch.mm(rows, _exact_unpack(s["w"][0][g], s["w"][1][g]).t())
                out[lo:lo + count] = _exact_act(c) if case["swiglu"] else c
                lo += count
        return out
    if op == "experts":
        x = _exact_block_values(s["x"])
        out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        for e, count in enumerate(s["counts"]):
            if count:
                token, slot = (s["idx"] == e).nonzero(as_tuple=True)
                act = _exact_act(torch.mm(x[token], _exact_unpack(s["gate_up"][0][e], s["gate_up"][1][e]).t()))
                y = torch.mm(_exact_block_values(act), _exact_unpack(s["down"][0][e], s["down"][1][e]).t())
                out[token] += y * s["weights"][token, slot].double().unsqueeze(1)
        return out
    y, res, w = s["y"].detach().double(), s["residual"].detach().double(), s["weight"].detach().double()
    t, h = y.shape
    eps, beta, alpha = s["eps"], s["branch_scale"], s["residual_scale"]
    gate = torch.ones(1, 1, dtype=torch.float64, device="cuda") if s["gate"] is None else s["gate"].detach().double()
    post = None if s["post_weight"] is None else s["post_weight"].detach().double()
    ry = 1.0 / torch.sqrt((y * y).sum(1, keepdim=True) / h + eps)
    z = y if post is None else y * ry * post
    hidden = alpha * res + beta * (gate * z)
    rh = 1.0 / torch.sqrt((hidden * hidden).sum(1, keepdim=True) / h + eps)
    out = {"hidden": hidden, "x": hidden * rh * w}
    if not case["train"]:
        return out
    gh, gx = s["d_hidden"].double(), s["d_x"].double()
    gw = gx * w
    dh = gh + rh * (gw - hidden * rh * rh * (gw * hidden).sum(1, keepdim=True) / h)
    dz = beta * gate * dh
    if post is None:
        out["d_y"] = dz
    else:
        out["d_y"] = ry * (dz * post - y * ry * ry * (dz * post * y).sum(1, keepdim=True) / h)
    out["d_residual"] = alpha * dh
    out["d_weight"] = (gx * hidden * rh).sum(0)
    if post is not None:
        out["d_post_weight"] = (dz * y * ry).sum(0)
    if s["gate"] is not None:
        dg = beta * dh * z
        out["d_gate"] = dg.sum(1, keepdim=True) if case["gate"] == "token" else dg.sum(0) if case["gate"] == "channel" else dg
    return out

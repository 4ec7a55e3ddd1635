"""residual_norm on the GPU: the residual sum with the norms, gate and scales around a block, and its gradients.

The oracle is the formula in float64.  Tolerances are counted, not fitted: u = 2^-24 is half a step of fp32, and
every value that the kernel forms carries the bound of its error along (class V).  A row sum adds at most 32 values
in a lane (31 sums), 6 levels of lanes and 3 more waves (16 values and 7 where eight waves share a row), so it is off
by at most 40 u of the sum of sizes; a column sum adds
ceil(T / walkers) rows in a walker, 64 to 256 walkers in a thread and 16 threads.  A product or sum of computed
values rounds once more; rsqrt is within 2 u and counts 4 with its argument.  The output rounds by 2^-8 (bf16) or
2^-24 (fp32) of the value.
"""

import pytest
import torch

from parallel_amd import residual_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


class V:
    """A float64 value and a bound on how far fp32 arithmetic may be from it."""

    def __init__(self, value, err=None):
        self.v, self.e = value, torch.zeros_like(value) if err is None else err

    @staticmethod
    def of(x):
        return x if isinstance(x, V) else V(torch.as_tensor(x, dtype=torch.float64, device=DEV))

    def __mul__(self, o):
        o = V.of(o)
        v = self.v * o.v
        e = self.e * (o.v.abs() + o.e) + self.v.abs() * o.e
        return V(v, e + (v.abs() + e) * U)

    def __add__(self, o):
        o = V.of(o)
        v = self.v + o.v
        e = self.e + o.e
        return V(v, e + (v.abs() + e) * U)

    def __neg__(self):
        return V(-self.v, self.e)

    def total(self, dim, depth):
        keep = dim == -1
        v = self.v.sum(dim, keepdim=keep)
        return V(v, self.e.sum(dim, keepdim=keep) * (1 + depth * U) + depth * U * self.v.abs().sum(dim, keepdim=keep))

    def rsqrt(self):
        v = self.v.rsqrt()
        return V(v, v * (0.5 * self.e / (self.v - self.e) * (1 + 1e-3) + 4 * U))


def oracle(y, residual, weight, post, gate, bs, rs, eps, d_hidden, d_x):
    """{name: V} of the outputs and gradients."""
    T, H = y.shape
    walkers = min(T, 4096 if H <= 512 else 1024)
    row, col = 40, -(-T // walkers) + (walkers + 15) // 16 + 16
    inv = 1.0 / H
    yv, rv, wv = (V(t.double()) for t in (y, residual, weight))
    bs, rs = (torch.tensor(float(torch.tensor(f, dtype=torch.float32)), dtype=torch.float64, device=DEV)
              for f in (bs, rs))  # the kernel's scales are floats
    eps = float(torch.tensor(eps, dtype=torch.float32))
    q = yv
    if post is not None:
        ry = ((yv * yv).total(-1, row) * inv + eps).rsqrt()
        q = yv * ry
    v = q if post is None else q * V(post.double())
    g = V(torch.ones(1, 1, dtype=torch.float64, device=DEV)) if gate is None else V(gate.double())
    h = rv * rs + (v * g) * bs
    r = ((h * h).total(-1, row) * inv + eps).rsqrt()
    out = {"hidden": h, "x": h * r * wv}
    dh = V(torch.zeros_like(h.v)) if d_hidden is None else V(d_hidden.double())
    out["weight"] = V(torch.zeros(H, dtype=torch.float64, device=DEV))
    if d_x is not None:
        dx = V(d_x.double())
        e = dx * wv
        k = r * r * r * inv * (e * h).total(-1, row)
        dh = dh + (r * e + -(k * h))
        out["weight"] = (dx * h * r).total(0, col)
    out["residual"] = dh * rs
    db = dh * bs
    dg = db * v
    dz = db * g
    if gate is not None:
        out["gate"] = dg.total(-1, row) if gate.shape == (T, 1) else dg.total(0, col) if gate.dim() == 1 else dg
    if post is None:
        out["y"] = dz
    else:
        f = dz * V(post.double())
        k = ry * ry * ry * inv * (f * yv).total(-1, row)
        out["y"] = ry * f + -(k * yv)
        out["post_weight"] = (dz * q).total(0, col)
    return out


def check(name, got, want):
    assert torch.isfinite(got).all(), name
    bound = want.v.abs() * HALF_STEP[got.dtype] + want.e * (1 + HALF_STEP[got.dtype]) + 1e-40
    off = (got.double() - want.v).abs()
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} of the bound, {float(off.max()):.3e} off"


def make(T, H, dtype, post, gate, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 131 * T + H)
    n = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    shape = {"none": None, "token": (T, 1), "channel": (H,), "full": (T, H)}[gate]
    t = dict(y=n(T, H), residual=2 * n(T, H), weight=1 + 0.2 * n(H), post_weight=1 + 0.2 * n(H) if post else None,
             gate=torch.sigmoid(n(*shape)) if shape else None)
    t = {k: None if v is None else v.to(dtype) for k, v in t.items()}
    return t, n(T, H).to(dtype), n(T, H).to(dtype)


def run(t, d_hidden, d_x, bs, rs, eps=1e-6):
    leaves = {k: v.detach().requires_grad_() for k, v in t.items() if v is not None}
    hidden, x = residual_norm(leaves["y"], leaves["residual"], leaves["weight"], post_weight=leaves.get("post_weight"),
                              gate=leaves.get("gate"), branch_scale=bs, residual_scale=rs, eps=eps)
    used = [(o, d) for o, d in ((hidden, d_hidden), (x, d_x)) if d is not None]
    grads = torch.autograd.grad([o for o, _ in used], list(leaves.values()), [d for _, d in used])
    return {"hidden": hidden.detach(), "x": x.detach(), **dict(zip(leaves, grads))}


def compare(t, d_hidden, d_x, bs, rs, eps=1e-6):
    got = run(t, d_hidden, d_x, bs, rs, eps)
    want = oracle(t["y"], t["residual"], t["weight"], t["post_weight"], t["gate"], bs, rs, eps, d_hidden, d_x)
    for name, value in got.items():
        check(name, value, want[name])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("post", [False, True], ids=["sum", "post"])
@pytest.mark.parametrize("gate", ["none", "token", "channel", "full"])
@pytest.mark.parametrize("T,H", [(1, 8), (5, 512), (3, 520), (7, 2048), (2, 2056), (3, 4104), (1, 8192)])
def test_outputs_and_gradients(T, H, gate, post, dtype):
    t, d_hidden, d_x = make(T, H, dtype, post, gate)
    compare(t, d_hidden, d_x, 0.22, 1.5)


@pytest.mark.parametrize("T,H,gate,post", [(4100, 72, "channel", True), (1030, 1024, "token", True),
                                           (2051, 4096, "none", False), (1500, 6000, "full", False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_more_rows_than_walkers(T, H, gate, post, dtype):
    t, d_hidden, d_x = make(T, H, dtype, post, gate)
    compare(t, d_hidden, d_x, 1.0, 1.0)


@pytest.mark.parametrize("T,H,gate", [(700, 4096, "token"), (600, 5008, "channel"), (600, 8192, "full"), (1, 8192, "token")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_several_wide_rows_per_walker_with_post(T, H, gate, dtype):
    t, d_hidden, d_x = make(T, H, dtype, True, gate)
    compare(t, d_hidden, d_x, 0.7, 1.2)


@pytest.mark.parametrize("gate,post,bs", [("none", False, 1.0), ("none", False, 0.5), ("token", True, 0.5)])
@pytest.mark.parametrize("which", ["hidden", "x"])
def test_one_output_alone_has_a_gradient(which, gate, post, bs):
    t, d_hidden, d_x = make(9, 264, torch.float32, post, gate)
    compare(t, d_hidden if which == "hidden" else None, d_x if which == "x" else None, bs, 1.0)


def test_rows_of_zeros_and_large_values():
    t, d_hidden, d_x = make(6, 256, torch.float32, True, "token")
    t["y"][0], t["residual"][1], t["gate"][2] = 0.0, 0.0, 0.0
    t["y"][3] *= 1e4
    t["residual"][4] *= 1e-4
    t["y"][5], t["residual"][5] = 0.0, 0.0  # the sum is zero too: rsqrt(eps) carries the row
    compare(t, d_hidden, d_x, 0.7, 1.0, eps=1e-5)


@pytest.mark.parametrize("post,gate", [(False, "none"), (True, "token"), (True, "channel"), (False, "full")])
def test_gradients_against_differences(post, gate):
    """<gradient, direction> against a central difference of the float64 formula along it."""
    t, d_hidden, d_x = make(5, 96, torch.float32, post, gate)
    got = run(t, d_hidden, d_x, 0.4, 1.1)
    want = oracle(t["y"], t["residual"], t["weight"], t["post_weight"], t["gate"], 0.4, 1.1, 1e-6, d_hidden, d_x)
    g = torch.Generator(device=DEV).manual_seed(5)

    def loss(name, step):
        s = {k: None if v is None else v.double() for k, v in t.items()}
        s[name] = s[name] + step
        o = oracle(s["y"], s["residual"], s["weight"], s["post_weight"], s["gate"], 0.4, 1.1, 1e-6, d_hidden, d_x)
        return float((o["hidden"].v * d_hidden.double()).sum() + (o["x"].v * d_x.double()).sum())

    for name, value in t.items():
        if value is None:
            continue
        along = torch.randn(value.shape, generator=g, device=DEV, dtype=torch.float64)
        eps = 1e-5
        slope = (loss(name, eps * along) - loss(name, -eps * along)) / (2 * eps)
        mine = float((got[name].double() * along).sum())
        # the kernel's bound along the direction; the difference's own error: its third derivative (of order one
        # per value here) times eps^2, and float64 cancellation 1e-16 / eps of a loss of some hundreds
        bound = float(((want[name].e + want[name].v.abs() * U) * along.abs()).sum()) + 1e-7 * (1 + abs(slope))
        assert abs(mine - slope) <= bound, (name, mine, slope, bound)


def test_strides_offsets_and_leading_dimensions():
    """Transposed, sliced, misaligned and expanded operands give what their contiguous copies do."""
    t, d_hidden, d_x = make(24, 64, torch.bfloat16, True, "token")
    want = run(t, d_hidden, d_x, 0.3, 1.0)
    odd = torch.empty(24 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(24, 64).copy_(t["y"])
    wide = torch.empty(24, 128, dtype=torch.bfloat16, device=DEV)[:, 32:96].copy_(t["residual"])
    turned = t["weight"].repeat(3, 1).t().contiguous().t()[1]
    s = dict(t, y=odd.view(2, 12, 64), residual=wide.unflatten(0, (2, 12)), weight=turned,
             gate=t["gate"].view(2, 12, 1))
    got = run(s, d_hidden.view(2, 12, 64), d_x.t().contiguous().t().view(2, 12, 64), 0.3, 1.0)
    for name, value in want.items():
        assert torch.equal(got[name].reshape(value.shape), value), name
    flat = t["gate"].expand(24, 64)  # a per-token gate given in full: its gradient comes back per element
    full = run(dict(t, gate=flat), d_hidden, d_x, 0.3, 1.0)
    assert full["gate"].shape == (24, 64) and torch.equal(full["x"], want["x"])


def test_no_rows():
    t, d_hidden, d_x = make(0, 64, torch.float32, True, "channel")
    got = run(t, d_hidden, d_x, 0.3, 1.0)
    assert got["hidden"].shape == got["x"].shape == (0, 64)
    for name in ("weight", "post_weight", "gate"):
        assert torch.equal(got[name], torch.zeros(64, device=DEV)), name


def test_the_same_bits_again_and_without_gradients():
    t, d_hidden, d_x = make(3000, 520, torch.bfloat16, True, "channel")
    a, b = run(t, d_hidden, d_x, 0.3, 1.0), run(t, d_hidden, d_x, 0.3, 1.0)
    for name, value in a.items():
        assert torch.equal(value, b[name]), name
    with torch.no_grad():
        hidden, x = residual_norm(t["y"], t["residual"], t["weight"], post_weight=t["post_weight"], gate=t["gate"],
                                  branch_scale=0.3)
    assert torch.equal(hidden, a["hidden"]) and torch.equal(x, a["x"])


def test_captured_forward_and_backward_replay_like_eager_calls():
    t, d_hidden, d_x = make(300, 1024, torch.bfloat16, True, "token")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        run(t, d_hidden, d_x, 0.3, 1.0)  # warm-up on the capture's kind of stream
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(t, d_hidden, d_x, 0.3, 1.0)
    for seed in range(3):
        new, nh, nx = make(300, 1024, torch.bfloat16, True, "token", seed=10 + seed)
        for name, value in new.items():
            t[name].copy_(value)
        d_hidden.copy_(nh)
        d_x.copy_(nx)
        graph.replay()
        torch.cuda.synchronize()
        want = run(t, d_hidden, d_x, 0.3, 1.0)
        for name, value in want.items():
            assert torch.equal(out[name], value), (seed, name)


def test_the_op_under_tracing_gives_the_same():
    """torch.library's own checks of the op: schema, fake kernel and autograd registration."""
    from parallel_amd import ops

    t, d_hidden, d_x = make(6, 64, torch.float32, True, "channel")
    args = (t["y"].requires_grad_(), t["residual"].requires_grad_(), t["weight"].requires_grad_(),
            t["post_weight"].requires_grad_(), t["gate"].requires_grad_(), 0.3, 1.0, 1e-6)
    torch.library.opcheck(torch.ops.parallel_amd.residual_norm_fwd.default, args,
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
    hidden, x, *_ = ops.residual_norm_fwd(*args)
    grads = torch.autograd.grad([hidden, x], args[:5], [d_hidden, d_x])
    plain = run({k: v.detach() for k, v in t.items()}, d_hidden, d_x, 0.3, 1.0)
    for name, value in zip(("y", "residual", "weight", "post_weight", "gate"), grads):
        assert torch.equal(value, plain[name]), name


def test_one_tensor_in_several_places():
    """y and residual the same leaf, the gate too, and one weight for both norms: the places' gradients add up."""
    t, d_hidden, d_x = make(37, 640, torch.float32, True, "full")
    t["residual"], t["gate"], t["post_weight"] = t["y"], t["y"], t["weight"]
    parts = run(t, d_hidden, d_x, 0.4, 1.1)
    y, w = t["y"].clone().requires_grad_(), t["weight"].clone().requires_grad_()
    hidden, x = residual_norm(y, y, w, post_weight=w, gate=y, branch_scale=0.4, residual_scale=1.1)
    torch.autograd.backward([hidden, x], [d_hidden, d_x])
    assert torch.equal(hidden, parts["hidden"]) and torch.equal(x, parts["x"])
    for got, names in ((y.grad, ("y", "residual", "gate")), (w.grad, ("weight", "post_weight"))):
        each = [parts[n].double() for n in names]
        bound = 2 * U * sum(e.abs() for e in each) * (1 + U)  # two fp32 sums, in any order
        assert ((got.double() - sum(each)).abs() <= bound).all()


def test_gradients_accumulate_apart_where_one_tensor_serves_two():
    """The plain sum's one gradient of y and residual: a second pass into .grad, and one changed in place."""
    t, d_hidden, d_x = make(24, 256, torch.float32, False, "none")
    once = run(t, d_hidden, d_x, 1.0, 1.0)
    leaves = [t[n].clone().requires_grad_() for n in ("y", "residual", "weight")]
    for _ in range(2):
        torch.autograd.backward(residual_norm(*leaves), [d_hidden, d_x])
    for leaf, name in zip(leaves, ("y", "residual", "weight")):
        assert torch.equal(leaf.grad, 2 * once[name]), name
    leaves[0].grad.zero_()
    assert torch.equal(leaves[1].grad, 2 * once["residual"])


def test_two_streams_and_two_graphs_at_once():
    cases = [make(700, 1024, torch.bfloat16, True, "channel", seed=s) for s in (1, 2)]
    want = [run(*c, 0.3, 1.0) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(run(*c, 0.3, 1.0))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for name in w:
                assert torch.equal(g[name], w[name]), name
    graphs, outs = [], []
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(*c, 0.3, 1.0))
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(outs, want):
            for name in w:
                assert torch.equal(g[name], w[name]), name


def test_rows_past_32_bits():
    """More than 2^31 values a tensor: the last rows as a call on them alone gives them."""
    T, H, tail = 270_000, 8192, 300
    assert T * H > 1 << 31
    block = torch.randn(1000, H, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).to(torch.bfloat16)
    big = lambda k: block.roll(k, 0).repeat(T // 1000, 1)  # noqa: E731
    y, residual, d_hidden, d_x = (big(k) for k in range(4))
    w, p = (1 + 0.1 * block[k] for k in range(2))
    t = dict(y=y, residual=residual, weight=w, post_weight=p, gate=block[:, :1].repeat(T // 1000, 1))
    got = run(t, d_hidden, d_x, 0.5, 1.0)
    last = {k: v if k in ("weight", "post_weight") else v[-tail:] for k, v in t.items()}
    want = run(last, d_hidden[-tail:], d_x[-tail:], 0.5, 1.0)
    for name in ("hidden", "x", "y", "residual", "gate"):
        assert torch.equal(got[name][-tail:], want[name]), name
    del got, want, y, residual, d_hidden, d_x, t, last
    torch.cuda.empty_cache()

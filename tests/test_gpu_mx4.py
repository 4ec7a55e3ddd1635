"""4-bit microscaled operands on the GPU: quantisation, the grouped products and the experts on them, against float64.

Codes, scales and their values must be equal.  The products' bounds are counted in mx4_oracle: fp32 accumulation,
then half a step of the bf16 output (2^-8); where act values are quantised on the way, a value that accumulation may
carry over a rounding border may take the neighbouring code, and counts with that distance.
"""

import pytest
import torch

import mx4_oracle as O
from parallel_amd import (
    MX4Experts,
    MX4Tensor,
    MoeConfig,
    SparseMoeBlock,
    mx4_experts,
    mx4_grouped_mm,
    mx4_swiglu,
    ops,
    quantize_mx4,
    residual_norm,
)
from parallel_amd._lib import call

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def pitch(K):
    return 8 * -(-K // 256)


def assert_quantized(x):
    q = quantize_mx4(x)
    idx, s = O.quantize(x)
    K = x.shape[-1]
    assert q.shape == x.shape and q.scales.shape == x.shape[:-1] + (pitch(K),)
    assert torch.equal(q.block_scales, s)
    assert torch.equal(q.codes, O.pack(idx))
    assert not q.scales[..., K // 32:].any()
    for dt in (torch.float32, BF):
        assert torch.equal(torch.nan_to_num(q.dequantize(dt).double(), nan=1e300),
                           torch.nan_to_num(O.values(idx, s).to(dt).double(), nan=1e300))
    return q


@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (7, 256), (5, 288), (2, 3, 640), (33, 2048), (1000, 160), (32,)])
def test_quantize_random(shape, dtype):
    g = gen(sum(shape))
    x = torch.randn(*shape, generator=g, device=DEV) * torch.exp(3 * torch.randn(*shape[:-1], 1, generator=g, device=DEV))
    assert_quantized(x.to(dtype))


def test_quantize_every_finite_bf16_value():
    """Every bf16 value in a block that its own size rules, and in one whose scale is up to 2^4 larger."""
    bits = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16)
    x = bits.view(BF)
    x = x[torch.isfinite(x)]
    own = x.view(-1, 1).expand(-1, 32).contiguous()
    assert_quantized(own)
    for up in (2.0, 4.0, 16.0):
        block = own.clone()
        block[:, 7] = (own[:, 7].double().abs() * up).clamp(max=3e38).to(BF)
        assert_quantized(block)


def test_quantize_at_rounding_borders():
    """fp32 values on and next to the middles between levels, at scales from the smallest to the largest."""
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], dtype=torch.float64, device=DEV)
    for e in (-127, -126, -100, -1, 0, 1, 60, 125):
        m = (mid * 2.0 ** e).float()
        if e > -120:  # neighbours; subnormal ones below that keep the borders themselves
            m = torch.cat((m, torch.nextafter(m, torch.full_like(m, 3e38)), torch.nextafter(m, -m)))
        x = torch.zeros(m.numel(), 32, device=DEV)
        x[:, 3] = 2.0 ** min(e + 2, 127)
        x[:, 5], x[:, 30] = m, -m
        assert_quantized(x)


def test_quantize_special_blocks():
    x = torch.randn(6, 96, generator=gen(3), device=DEV)
    x[0, 40], x[1, 64], x[2, 0] = float("nan"), float("inf"), -float("inf")
    x[3] = 0.0
    x[4, 32:64] = -0.0
    x[5, :32] = 3.4e38
    for dt in (torch.float32, BF):
        q = assert_quantized(x.to(dt))
        assert q.block_scales[0].tolist()[1] == 255 and torch.isnan(q.dequantize()[0, 32:64]).all()
        assert torch.isfinite(q.dequantize()[0, :32]).all()
    assert_quantized(torch.full((2, 32), 1e-45, device=DEV))  # fp32 subnormals
    assert quantize_mx4(torch.empty(0, 64, device=DEV)).dequantize().shape == (0, 64)


def test_every_code_at_every_scale_dequantizes_exactly():
    codes = torch.arange(256, device=DEV, dtype=torch.int32).to(torch.uint8).view(256, 1).expand(256, 16).contiguous()
    codes = torch.cat((codes[:128], codes[128:]), dim=1)  # [128, 32]: two blocks a row
    for s in range(256):
        scales = torch.zeros(128, 8, dtype=torch.uint8, device=DEV)
        scales[:, 0], scales[:, 1] = s, 255 - s
        t = MX4Tensor(codes, scales)
        want = O.values(O.unpack(codes), scales)
        for dt in (torch.float32, BF):
            got = t.dequantize(dt)
            assert torch.equal(torch.isnan(got), torch.isnan(want)), s
            assert torch.equal(torch.nan_to_num(got.double(), nan=0.0, posinf=1e300, neginf=-1e300),
                               torch.nan_to_num(want.to(dt).double(), nan=0.0, posinf=1e300, neginf=-1e300)), s


def operand(g, *shape, std=1.0):
    """(MX4Tensor, its float64 values) of random codes from normal data."""
    x = torch.randn(*shape, generator=g, device=DEV) * std
    x = x * torch.exp(0.7 * torch.randn(*shape[:-2], 1, shape[-1], generator=g, device=DEV))
    idx, s = O.quantize(x)
    scales = torch.full(shape[:-1] + (pitch(shape[-1]),), 255, dtype=torch.uint8, device=DEV)  # padding is never read as NaN
    scales[..., :s.shape[-1]] = s
    return MX4Tensor(O.pack(idx), scales), O.values(idx, s)


def within(got, want, err, what=""):
    bound = want.abs() * 2.0 ** -8 + err * (1 + 2.0 ** -8) + 1e-38
    off = (got.double() - want).abs()
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"


def offsets_of(counts):
    return torch.tensor(counts, dtype=torch.int32, device=DEV).cumsum(0, dtype=torch.int32)


COUNTS = [
    [1], [0, 3], [5, 0, 0, 1], [16, 17], [1] * 40, [63, 64, 65, 0], [130, 2, 0, 33], [0] * 70 + [9] + [0] * 20 + [1],
    [300, 129], [256, 257, 511], [1100],
]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("N,K", [(8, 32), (40, 96), (200, 544), (264, 2080)])
def test_grouped_products(counts, N, K):
    g = gen(N + K + sum(counts))
    a, av = operand(g, sum(counts), K)
    w, wv = operand(g, len(counts), 2 * N, K, std=0.1)
    offs = offsets_of(counts)
    want, err = O.product(av, wv, counts)
    within(mx4_grouped_mm(a, w, offs), want, err, "mm")
    act, e = O.swiglu(want, err)
    within(mx4_swiglu(a, w, offs), act, e, "swiglu")


# Mean rows for each kernel: few rows in all; 64-, 128- and 256-row tiles; K with an odd number of 256-value stages,
# with part of one, and with one; columns past a tile; one or two rows in most tiles; one group with nearly all rows.
@pytest.mark.parametrize("rows,G,N,K,skew", [
    (40, 5, 200, 544, 0), (2000, 64, 328, 544, 0), (384, 128, 264, 512, 0), (2600, 64, 520, 96, 0), (1500, 64, 520, 1056, 2),
    (1000, 8, 328, 544, 0), (1300, 10, 264, 800, 0), (900, 8, 136, 32, 0), (2000, 8, 328, 544, 0), (900, 3, 264, 2080, 0),
    (5000, 16, 264, 288, 2), (700, 2, 8, 256, 0), (4096, 300, 264, 160, 0),
])
def test_every_tile_height(rows, G, N, K, skew):
    g = gen(rows + K)
    weight = (torch.arange(G, device=DEV) + 1.0) ** -float(skew)
    counts = torch.bincount(torch.multinomial(weight, rows, replacement=True, generator=g), minlength=G).tolist()
    a, av = operand(g, rows, K)
    w, wv = operand(g, G, 2 * N, K, std=0.1)
    want, err = O.product(av, wv, counts)
    within(mx4_grouped_mm(a, w, offsets_of(counts)), want, err, "mm")
    within(mx4_swiglu(a, w, offsets_of(counts)), *O.swiglu(want, err), "swiglu")


@pytest.mark.parametrize("rows,G,N,K", [(3000, 8, 512, 768), (700, 3, 768, 1024), (9000, 64, 256, 256), (130, 128, 96, 1536)])
def test_larger_products(rows, G, N, K):
    g = gen(rows)
    counts = torch.bincount(torch.randint(G, (rows,), generator=g, device=DEV), minlength=G).tolist()
    a, av = operand(g, rows, K)
    w, wv = operand(g, G, 2 * N, K, std=0.1)
    want, err = O.product(av, wv, counts)
    within(mx4_grouped_mm(a, w, offsets_of(counts)), want, err, "mm")
    within(mx4_swiglu(a, w, offsets_of(counts)), *O.swiglu(want, err), "swiglu")


# Sizes whose passes over 256 CUs take 128-row tiles (K over 1024; 16 tiles down by 16 across), 256-row tiles (16 by 16
# of those), and the few-row kernel for many rows of a narrow product; whole and broken stages of K, groups with a row or none.
@pytest.mark.parametrize("rows,N", [(2000, 2000), (1990, 1928), (4000, 2000), (4090, 1928), (4096, 40), (1500, 96)])
@pytest.mark.parametrize("K,counts", [(1056, [0.5, 0.0, 0.3, 0.2]), (2048, [1.0]), (32, [1.0]), (544, [0.3, 0.0, 0.001, 0.6]), (768, [1 / 9] * 9), (288, [0.0, 0.97, 0.0, 0.001])])
def test_passes_over_the_card(rows, N, K, counts):
    counts = [int(c * rows) for c in counts]
    rows = sum(counts)
    g = gen(rows + K)
    a, av = operand(g, rows, K)
    w, wv = operand(g, len(counts), 2 * N, K, std=0.1)
    want, err = O.product(av, wv, counts)
    within(mx4_grouped_mm(a, w, offsets_of(counts)), want, err, "mm")
    within(mx4_swiglu(a, w, offsets_of(counts)), *O.swiglu(want, err), "swiglu")


def test_nan_blocks_reach_their_rows_and_columns_alone():
    g = gen(8)
    counts = [20, 0, 50]
    a, av = operand(g, 70, 320)
    w, wv = operand(g, 3, 48, 320)
    a.scales[33, 4] = 255
    w.scales[0, 5, 9] = 255
    av[33, 128:160] = float("nan")
    wv[0, 5, 288:] = float("nan")
    got = mx4_grouped_mm(a, w, offsets_of(counts))
    want, _ = O.product(av, wv, counts)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert bool(torch.isnan(want[33]).all()) and int(torch.isnan(want).sum()) == 48 + 20 - 0


@pytest.mark.parametrize("rows,counts", [(50, [10, 0, 20]), (600, [100, 257]), (40, [0, 0, 0]), (9, [0, 9])])
def test_rows_behind_the_last_group_are_left_as_they_were(rows, counts):
    g = gen(rows)
    G, N, K, used = len(counts), 72, 288, sum(counts)
    a, av = operand(g, rows, K)
    w, wv = operand(g, G, 2 * N, K)
    offs = offsets_of(counts)
    s = torch.cuda.current_stream().cuda_stream
    c = torch.full((rows, 2 * N), 7.0, dtype=BF, device=DEV)
    call("moe_mx4_grouped_gemm", a.codes.data_ptr(), a.scales.data_ptr(), rows, None, 1, w.codes.data_ptr(),
         w.scales.data_ptr(), offs.data_ptr(), G, rows, 2 * N, K, c.data_ptr(), s)
    want, err = O.product(av[:used], wv, counts)
    within(c[:used], want, err)
    assert bool((c[used:] == 7.0).all())
    w32, wv32 = operand(g, G, 64, K)
    codes = torch.full((rows, 16), 0x5a, dtype=torch.uint8, device=DEV)
    scales = torch.full((rows, 8), 0x33, dtype=torch.uint8, device=DEV)
    call("moe_mx4_grouped_swiglu", a.codes.data_ptr(), a.scales.data_ptr(), rows, None, 1, w32.codes.data_ptr(),
         w32.scales.data_ptr(), offs.data_ptr(), G, rows, 32, K, None, codes.data_ptr(), scales.data_ptr(), s)
    act, e = O.swiglu(*O.product(av[:used], wv32, counts))
    mid, far = O.requantize(act, e)
    assert bool(((O.values(O.unpack(codes[:used]), scales[:used]) - mid).abs() <= far).all())
    assert bool((codes[used:] == 0x5a).all()) and bool((scales[used:] == 0x33).all())


def layer(g, E, H, I):
    gu, guv = operand(g, E, 2 * I, H, std=H ** -0.5)
    dn, dnv = operand(g, E, H, I, std=I ** -0.5)
    return gu, guv, dn, dnv


def experts_oracle(x, idx, wts, guv, dnv):
    """(out, bound) of the path: quantised tokens, fp32 products, quantised act, fp32 or bf16 rows, fp32 combine."""
    E = guv.shape[0]
    xv = O.values(*O.quantize(x))
    T, k = idx.shape
    out, err = torch.zeros(T, x.shape[1], dtype=torch.float64, device=DEV), None
    err, size = torch.zeros_like(out), torch.zeros_like(out)
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        act, ea = O.swiglu(*O.product(xv[t], guv[e:e + 1], [t.numel()]))
        mid, far = O.requantize(act, ea)
        y, ey = O.product(mid, dnv[e:e + 1], [t.numel()])
        ey = ey + far @ dnv[e].t().abs()
        if x.dtype == BF and x.shape[0] * k * x.shape[1] > 1 << 22:  # the rows are held in bf16
            ey = ey + 2.0 ** -8 * (y.abs() + ey)
        wt = wts[t, j].double().unsqueeze(1)
        out.index_add_(0, t, wt * y)
        err.index_add_(0, t, wt.abs() * ey)
        size.index_add_(0, t, (wt * y).abs())
    return out, err + 2 * k * O.U * (size + err)


@pytest.mark.parametrize("T,H,E,k,I", [(1, 64, 8, 2, 32), (1, 2048, 128, 8, 768), (7, 256, 8, 2, 128), (48, 512, 32, 4, 160),
                                       (333, 416, 8, 3, 288), (1500, 512, 4, 2, 256), (4096, 256, 16, 2, 96),
                                       (8, 256, 16, 8, 64), (9, 256, 16, 8, 64), (3, 288, 32, 16, 1312), (21, 1056, 8, 3, 96), (300, 256, 32, 4, 288),
                                       (100, 512, 64, 4, 320), (3000, 512, 8, 4, 64), (2500, 1056, 64, 2, 160)])
def test_experts(T, H, E, k, I):
    g = gen(T + H)
    gu, guv, dn, dnv = layer(g, E, H, I)
    x = (torch.randn(T, H, generator=g, device=DEV) * 2).to(BF)
    top = torch.topk(torch.randn(T, E, generator=g, device=DEV), k, dim=1)
    wts = torch.softmax(top.values, 1)
    within(mx4_experts(x, top.indices, wts, gu, dn), *experts_oracle(x, top.indices, wts, guv, dnv))


# Slots in their own order or sorted: 128 and 130 of them, many that share few experts of small and of large weights,
# more choices than experts.
@pytest.mark.parametrize("T,H,E,k,I", [(16, 256, 64, 8, 96), (13, 256, 64, 10, 96), (64, 512, 4, 2, 256), (16, 2048, 4, 2, 2048),
                                       (2, 2048, 4, 2, 2048), (1, 4096, 4, 4, 2048), (128, 64, 1, 1, 32)])
@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "fp32"])
def test_experts_of_few_slots(T, H, E, k, I, dtype):
    g = gen(T + H + E)
    gu, guv, dn, dnv = layer(g, E, H, I)
    x = (torch.randn(T, H, generator=g, device=DEV) * 2).to(dtype)
    top = torch.topk(torch.randn(T, E, generator=g, device=DEV), k, dim=1)
    wts = torch.softmax(top.values, 1)
    within(mx4_experts(x, top.indices, wts, gu, dn), *experts_oracle(x, top.indices, wts, guv, dnv))


def test_experts_with_more_choices_than_experts():
    g = gen(9)
    gu, guv, dn, dnv = layer(g, 2, 128, 64)
    x = torch.randn(5, 128, generator=g, device=DEV).to(BF)
    idx = torch.randint(2, (5, 6), generator=g, device=DEV)
    wts = torch.rand(5, 6, generator=g, device=DEV)
    within(mx4_experts(x, idx, wts, gu, dn), *experts_oracle(x, idx, wts, guv, dnv))


# The same with the act values quantised and the rows of down in bf16 (bf16 hidden states of this size) and fp32.
@pytest.mark.parametrize("T", [500, 1013])
@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "fp32"])
def test_experts_on_tall_tiles(T, dtype):
    E, H, k, I = 6, 4000, 4, 1984
    g = gen(T)
    gu, guv, dn, dnv = layer(g, E, H, I)
    x = (torch.randn(T, H, generator=g, device=DEV) * 2).to(dtype)
    top = torch.topk(torch.randn(T, E, generator=g, device=DEV) - torch.arange(E, device=DEV) * 0.5, k, dim=1)
    wts = torch.softmax(top.values, 1)
    within(mx4_experts(x, top.indices, wts, gu, dn), *experts_oracle(x, top.indices, wts, guv, dnv))


def test_experts_routing_corners():
    """Sentinel ids, a token without any expert, the same expert twice for a token, all tokens on one expert,
    weights of zero, fp32 hidden states, int32 ids."""
    g = gen(4)
    E, H, I, T = 8, 128, 64, 70
    gu, guv, dn, dnv = layer(g, E, H, I)
    x = torch.randn(T, H, generator=g, device=DEV)
    idx = torch.full((T, 3), 5, device=DEV)
    idx[10:30, 0] = E  # the sentinel
    idx[20, :] = E
    idx[40:, 1] = torch.randint(E, (30,), generator=g, device=DEV)
    wts = torch.rand(T, 3, generator=g, device=DEV)
    wts[3] = 0.0
    for dt in (torch.float32, BF):
        out = mx4_experts(x.to(dt), idx.int(), wts, gu, dn)
        assert out.dtype == dt
        within(out, *experts_oracle(x.to(dt), idx, wts, guv, dnv))
        assert not out[20].any() and not out[3].any()
    few = slice(15, 35)  # few enough slots to go without a sort, with sentinels and repeated experts among them
    for dt in (torch.float32, BF):
        out = mx4_experts(x[few].to(dt), idx[few], wts[few], gu, dn)
        assert out.dtype == dt and not out[5].any()
        within(out, *experts_oracle(x[few].to(dt), idx[few], wts[few], guv, dnv))
    neg = idx[few].clone()
    neg[3, 1] = -1
    out = mx4_experts(x[few], neg, wts[few], gu, dn)
    within(out, *experts_oracle(x[few], neg, wts[few], guv, dnv))
    x[6, 17] = float("inf")
    few = mx4_experts(x[:9], idx[:9], wts[:9], gu, dn)
    assert torch.isnan(few[6]).all() and torch.isfinite(few[:6]).all() and torch.isfinite(few[7:]).all()
    bad = mx4_experts(x, idx, wts, gu, dn)
    assert torch.isnan(bad[6]).all() and torch.isfinite(bad[torch.arange(T, device=DEV) != 6]).all()
    assert mx4_experts(x[:0], idx[:0], wts[:0], gu, dn).shape == (0, H)


def test_strided_and_misaligned_operands():
    g = gen(12)
    a, _ = operand(g, 40, 256)
    w, _ = operand(g, 2, 64, 256)
    offs = offsets_of([13, 27])
    want = mx4_grouped_mm(a, w, offs)
    codes = torch.empty(40 * 128 + 1, dtype=torch.uint8, device=DEV)[1:].view(40, 128).copy_(a.codes)
    scales = torch.empty(40, 24, dtype=torch.uint8, device=DEV)[:, 3:11].copy_(a.scales)
    turned = MX4Tensor(w.codes.transpose(0, 1).contiguous().transpose(0, 1), w.scales.flip(0).flip(0))
    every_other = torch.stack((offs, offs), 1).reshape(-1)[::2]
    assert torch.equal(mx4_grouped_mm(MX4Tensor(codes, scales), turned, every_other), want)
    x = torch.randn(256, 64, generator=g, device=DEV).to(BF)
    assert torch.equal(quantize_mx4(x.t()).codes, quantize_mx4(x.t().contiguous()).codes)
    unpadded = MX4Tensor(a.codes[:, :48].contiguous(), a.scales[:, :3].contiguous())  # K = 96: 3 bytes a row given
    assert unpadded.scales.shape == (40, 8) and unpadded.shape == (40, 96)


def test_replays_of_a_captured_layer_and_another_stream():
    g = gen(21)
    E, H, I, T = 16, 256, 128, 37
    gu, _, dn, _ = layer(g, E, H, I)
    x = torch.randn(T, H, generator=g, device=DEV).to(BF)
    top = torch.topk(torch.randn(T, E, generator=g, device=DEV), 4, dim=1)
    idx, wts = top.indices.clone(), torch.softmax(top.values, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = mx4_experts(x, idx, wts, gu, dn)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, mx4_experts(x, idx, wts, gu, dn))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mx4_experts(x, idx, wts, gu, dn)
    for n in range(3):
        x.copy_(torch.randn(T, H, generator=g, device=DEV))
        idx.copy_(torch.topk(torch.randn(T, E, generator=g, device=DEV), 4, dim=1).indices)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mx4_experts(x, idx, wts, gu, dn)), n


@pytest.mark.parametrize("rows,K", [(4097, 8192), (33000, 1056)])
@pytest.mark.parametrize("dtype", [BF, torch.float32], ids=["bf16", "fp32"])
def test_large_tensors_to_codes_and_back(rows, K, dtype):
    """More than 2^25 values, the last threads' chunks in part past the end: each row as it is in a small tensor."""
    x = torch.randn(rows, K, generator=gen(rows), device=DEV).to(dtype)
    assert x.numel() > 1 << 25
    q = quantize_mx4(x)
    back = q.dequantize(dtype)
    for lo in (0, rows // 2, rows - 70):
        part = assert_quantized(x[lo:lo + 70])
        assert torch.equal(q.codes[lo:lo + 70], part.codes) and torch.equal(q.scales[lo:lo + 70], part.scales)
        assert torch.equal(back[lo:lo + 70], part.dequantize(dtype))


def test_two_streams_and_two_graphs_at_once():
    g = gen(22)
    E, H, I = 32, 512, 256
    gu, _, dn, _ = layer(g, E, H, I)
    cases = []
    for T in (5, 7, 600):  # two without the sort, one with
        top = torch.topk(torch.randn(T, E, generator=g, device=DEV), 4, dim=1)
        cases.append((torch.randn(T, H, generator=g, device=DEV).to(BF), top.indices, torch.softmax(top.values, 1)))
    want = [mx4_experts(*c, gu, dn) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(mx4_experts(*c, gu, dn))
        torch.cuda.synchronize()
        assert all(map(torch.equal, got, want))
    graphs, outs = [], []
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(mx4_experts(*c, gu, dn))
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(map(torch.equal, outs, want))


def test_values_past_32_bits():
    """Quantisation of more than 2^31 values, weights of more than 2^31 bytes of codes, products and experts with more
    than 2^31 outputs: the last part as a call on it alone gives it."""
    g = gen(23)
    block, other = (torch.randn(1024, 4096, generator=g, device=DEV).to(BF) for _ in range(2))
    x = block.repeat(520, 1)
    x[-1024:] = other
    assert x.numel() > 1 << 31
    q, part = quantize_mx4(x), quantize_mx4(other)
    assert torch.equal(q.codes[-1024:], part.codes) and torch.equal(q.scales[-1024:], part.scales)
    assert torch.equal(q.dequantize()[-1024:], part.dequantize())
    del x

    w = MX4Tensor(q.codes.view(260, 2048, 2048).repeat(2, 1, 1), q.scales.view(260, 2048, 128).repeat(2, 1, 1))
    assert w.codes.numel() > 1 << 31
    tail, tailv = operand(g, 8, 2048, 4096, std=0.1)
    w.codes[-8:], w.scales[-8:] = tail.codes, tail.scales
    a, av = operand(g, 520, 4096)
    each = torch.arange(1, 521, dtype=torch.int32, device=DEV)  # a row a group
    want, err = O.product(av[-8:], tailv, [1] * 8)
    within(mx4_grouped_mm(a, w, each)[-8:], want, err, "mm")
    within(mx4_swiglu(a, w, each)[-8:], *O.swiglu(want, err), "swiglu")
    del w, q

    rows = 1_100_000
    a = MX4Tensor(part.codes[:, :64].repeat(rows // 1000, 1)[:rows], part.scales[:, :8].repeat(rows // 1000, 1)[:rows])
    w, _ = operand(g, 2, 2048, 128)
    offs = offsets_of([rows - 5000, 5000])
    out = mx4_grouped_mm(a, w, offs)
    assert out.numel() > 1 << 31
    last = MX4Tensor(a.codes[-5000:].contiguous(), a.scales[-5000:].contiguous())
    assert torch.equal(out[-5000:], mx4_grouped_mm(last, w, offsets_of([0, 5000])))
    del out, a

    T, E, H, I, k = 140_000, 16, 2048, 64, 8
    assert T * k * H > 1 << 31
    gu, _, dn, _ = layer(g, E, H, I)
    x = block[:, :H].repeat(140, 1)[:T].contiguous()
    idx = torch.topk(torch.randn(T, E, generator=g, device=DEV), k, dim=1).indices
    wts = torch.rand(T, k, generator=g, device=DEV)
    out = mx4_experts(x, idx, wts, gu, dn)
    tail = 4000  # (rows of down in bf16 for it too)
    assert torch.equal(out[-tail:], mx4_experts(x[-tail:], idx[-tail:], wts[-tail:], gu, dn))
    del out, x
    torch.cuda.empty_cache()


def test_modules_run_together_between_two_blocks():
    """Residual norm, router, experts on 4-bit weights, residual norm: the layer's second half as inference runs it."""
    g = gen(30)
    cfg = MoeConfig(hidden_size=256, num_experts=16, num_experts_per_tok=4, moe_intermediate_size=96, norm_topk_prob=True)
    block = SparseMoeBlock(cfg).to(DEV, BF)
    with torch.no_grad():
        for p in block.parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=DEV) * 0.06)
        block.experts = MX4Experts.from_experts(block.experts)
        attn, stream = (torch.randn(2, 45, 256, generator=g, device=DEV).to(BF) for _ in range(2))
        n1, n2 = (1 + 0.1 * torch.randn(256, generator=g, device=DEV).to(BF) for _ in range(2))
        hidden, x = residual_norm(attn, stream, n1)
        moe = block(x)
        out, nxt = residual_norm(moe, hidden, n2)
        _, scores, idx = block.gate(x.view(-1, 256))
    ex = block.experts
    values = [O.values(O.unpack(c), s) for c, s in ((ex.gate_up_codes, ex.gate_up_scales), (ex.down_codes, ex.down_scales))]
    within(moe.view(-1, 256), *experts_oracle(x.view(-1, 256), idx, scores, *values), "experts")
    h = hidden.double() + moe.double()
    assert bool(((out.double() - h).abs() <= h.abs() * 2.0 ** -8 + 4 * O.U * (hidden.double().abs() + moe.double().abs())).all())
    want = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * n2.double()
    assert bool(((nxt.double() - want).abs() <= want.abs() * (2.0 ** -8 + 64 * O.U) + 1e-6).all())
    state = block.state_dict()
    other = SparseMoeBlock(cfg).to(DEV, BF)
    other.experts = MX4Experts(*(MX4Tensor(torch.zeros_like(c), torch.zeros_like(s))
                                 for c, s in ((ex.gate_up_codes, ex.gate_up_scales), (ex.down_codes, ex.down_scales))))
    other.load_state_dict(state)
    with torch.no_grad():
        assert torch.equal(other(x), moe)


def test_a_transformers_block_takes_the_module():
    modeling = pytest.importorskip("transformers.models.qwen3_moe.modeling_qwen3_moe")
    from transformers import Qwen3MoeConfig

    cfg = Qwen3MoeConfig(hidden_size=128, num_experts=8, num_experts_per_tok=2, moe_intermediate_size=64,
                         norm_topk_prob=True)
    block = modeling.Qwen3MoeSparseMoeBlock(cfg).to(DEV, BF)
    g = gen(31)
    with torch.no_grad():
        for p in block.parameters():
            p.copy_(torch.randn(p.shape, generator=g, device=DEV) * 0.1)
        x = torch.randn(1, 20, 128, generator=g, device=DEV).to(BF)
        block.experts = MX4Experts.from_experts(block.experts)
        out = block(x)
        out = out[0] if isinstance(out, tuple) else out
        flat = x.view(-1, 128)
        gate = block.gate(flat)
        want = block.experts(flat, gate[2], gate[1])
    assert torch.equal(out.view(-1, 128), want)


def test_gradients_are_refused():
    g = gen(1)
    gu, _, dn, _ = layer(g, 4, 64, 32)
    x = torch.randn(3, 64, generator=g, device=DEV).to(BF).requires_grad_()
    idx = torch.zeros(3, 1, dtype=torch.int64, device=DEV)
    for call_it in (lambda: quantize_mx4(x), lambda: mx4_experts(x, idx, torch.ones(3, 1, device=DEV), gu, dn)):
        with pytest.raises(ValueError, match="no gradient"):
            call_it()
        with torch.no_grad():
            call_it()


def test_the_ops_pass_torch_library_checks():
    g = gen(2)
    gu, _, dn, _ = layer(g, 4, 64, 32)
    x = torch.randn(5, 64, generator=g, device=DEV).to(BF)
    idx = torch.randint(4, (5, 2), generator=g, device=DEV)
    a = quantize_mx4(x)
    offs = offsets_of([2, 0, 3, 0])
    lib = torch.ops.parallel_amd
    for op, args in ((lib.mx4_quantize, (x,)), (lib.mx4_dequantize, (a.codes, a.scales, True)),
                     (lib.mx4_grouped_mm, (a.codes, a.scales, gu.codes, gu.scales, offs)),
                     (lib.mx4_grouped_swiglu, (a.codes, a.scales, gu.codes, gu.scales, offs)),
                     (lib.mx4_experts, (x, idx, torch.ones(5, 2, device=DEV), gu.codes, gu.scales, dn.codes, dn.scales))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))

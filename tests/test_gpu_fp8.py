"""GPU parity of the 8-bit expert operators: block quantisation bit by bit, the grouped GEMM of
such operands against its 64-bit definition.

Tolerances of the GEMM, for an output of K products with S = sum |a b|:
  accumulation in fp32, any order: K * 2^-24 * S;
  rounding to bf16: half a step, 2^-8 of the value; to e4m3: 2^-4 of the value, or 2^-10 of the
  scale below the normal range.
"""
import numpy as np
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu

KINDS = ("normal", "zeros", "tiny", "huge", "edge", "nonfinite")


def _matrix(kind, m, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    if kind == "zeros":
        x[: max(1, m // 2)] = 0
        x[:, : k // 2] = -0.0
    elif kind == "tiny":  # subnormal blocks beside blocks of the smallest normal numbers
        x = x * 2.0 ** -126
        x[::2] *= 2.0 ** -9
    elif kind == "huge":
        x = x.clamp(-3, 3) * 2.0 ** 126
    elif kind == "edge":  # amax at and next to 448 * 2^e, values half-way between two e4m3 numbers
        x = torch.randint(-16, 17, (m, k), generator=g).float() / 16 * 1.0625
        x[:, 0] = 448.0
        if m > 1:
            x[1::2, 0] = 449.0 if dtype == torch.float32 else 450.0
    elif kind == "nonfinite":
        x[0, 0] = float("inf")
        x[-1, -1] = float("nan")
        x[m // 2, k // 2] = -float("inf")
        if m > 2:
            x[2] = float("nan")
    return x.to(dtype)


def _check_quantised(q, want_q, want_s):
    assert torch.equal(ref.bytes_of(q.scale.cpu()), want_s)
    got, want = q.data.cpu().float(), want_q.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = torch.where(torch.isnan(want), torch.zeros_like(want), want)
    assert torch.equal(torch.where(torch.isnan(got), torch.zeros_like(got), got), same)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k", [(1, 16), (3, 128), (5, 144), (37, 2064), (130, 7168)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_rows(cuda_dev, kind, m, k, dtype):
    import moe_b200
    x = _matrix(kind, m, k, dtype, m + k)
    _check_quantised(moe_b200.quantize_fp8(x.to(cuda_dev)), *ref.quantize(x, True))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("g,n,k", [(1, 1, 16), (2, 129, 144), (3, 300, 1040), (1, 128, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_weight(cuda_dev, kind, g, n, k, dtype):
    import moe_b200
    w = torch.stack([_matrix(kind, n, k, dtype, 7 * i + n) for i in range(g)])
    _check_quantised(moe_b200.quantize_fp8_weight(w.to(cuda_dev)), *ref.quantize(w, False))


def test_quantize_views_and_empty(cuda_dev):
    import moe_b200
    x = _matrix("normal", 64, 256, torch.bfloat16, 1).to(cuda_dev)
    for v in (x.t()[16:], x[:, 16:144], x[1:, :], x.flatten()[1:-15].view(-1, 16)):
        q = moe_b200.quantize_fp8(v)
        _check_quantised(q, *ref.quantize(v.cpu(), True))
    q = moe_b200.quantize_fp8(x[:0])
    assert q.data.shape == (0, 256) and q.scale.shape == (0, 2)
    assert moe_b200.quantize_fp8_weight(x.view(2, 32, 256)[:0]).scale.shape == (0, 1, 2)
    assert moe_b200.dequantize_fp8(q).shape == (0, 256)


@pytest.mark.parametrize("m,k", [(1, 16), (33, 144), (300, 2048)])
def test_dequantize(cuda_dev, m, k):
    """Every e4m3 code under small, large and special scales; exact in bf16."""
    import moe_b200
    g = torch.Generator().manual_seed(k)
    data = torch.randint(0, 256, (m, k), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sb = torch.randint(10, 240, (m, -(-k // 128)), generator=g, dtype=torch.uint8)
    sb[0, 0] = 0
    if m > 2:
        sb[1, 0], sb[2, 0] = 255, 1
    got = moe_b200.dequantize_fp8(moe_b200.Fp8Tensor(
        data.to(cuda_dev), sb.view(torch.float8_e8m0fnu).to(cuda_dev))).cpu()
    s = torch.where(sb == 255, torch.tensor(float("nan"), dtype=torch.float64),
                    torch.exp2(sb.double() - 127)).repeat_interleave(128, 1)[:, :k]
    want = data.double() * s
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.equal(got[ok], want[ok].to(torch.bfloat16))


@pytest.mark.parametrize("t,h,e,k", [(1, 16, 4, 1), (9, 144, 8, 3), (257, 2048, 64, 8),
                                     (64, 7168, 320, 8), (40, 256, 32, 32)])
def test_permute_fp8(cuda_dev, t, h, e, k):
    """Equal to quantising and then permuting, untouched rows and bad entries included."""
    import moe_b200
    g = torch.Generator().manual_seed(t + h)
    x = _matrix("normal", t, h, torch.bfloat16, h).to(cuda_dev)
    idx = torch.rand(t, e, generator=g).argsort(1)[:, :k].contiguous().to(cuda_dev)
    on = torch.zeros(t, e, dtype=torch.bool, device=cuda_dev).scatter_(1, idx, True)
    rim = moe_b200.row_id_map(on)
    q = moe_b200.permute_fp8(x, rim.map_te, idx, t * k)
    want = moe_b200.quantize_fp8(x)
    dst = rim.map_te.gather(1, idx)
    assert torch.equal(ref.bytes_of(q.data)[dst], ref.bytes_of(want.data)[:, None].expand(-1, k, -1))
    assert torch.equal(ref.bytes_of(q.scale)[dst], ref.bytes_of(want.scale)[:, None].expand(-1, k, -1))
    # entries that name no expert or no row are skipped
    bad = idx.clone()
    bad[0, 0], bad[-1, -1] = -1, e
    short = max(1, t * k - 2)
    q2 = moe_b200.permute_fp8(x, rim.map_te, bad, short)
    ok = (bad >= 0) & (bad < e)
    ok &= dst < short
    assert torch.equal(ref.bytes_of(q2.data)[dst[ok]], ref.bytes_of(q.data)[dst[ok]])


# ------------------------------------------------------------------------------------------- GEMM
def _operands(dev, rows, g, n, k, layout, seed, std=0.05):
    import moe_b200
    gen = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, k, generator=gen, device=dev)
    x *= torch.exp2(torch.randint(-4, 5, (rows, 1), generator=gen, device=dev).float())
    shape = (g, n, k) if layout == "NK" else (g, k, n)
    w = torch.randn(shape, generator=gen, device=dev) * std
    w *= torch.exp2(torch.randint(-3, 4, (g, 1, 1), generator=gen, device=dev).float())
    return moe_b200.quantize_fp8(x), moe_b200.quantize_fp8_weight(w)


def _product64(x, w, splits, layout):
    """(product, sum of magnitudes) in 64 bits; rows in no group are NaN."""
    xv = ref.values(x.data, ref.bytes_of(x.scale), True)
    wv = ref.values(w.data, ref.bytes_of(w.scale), False)
    n = wv.shape[1] if layout == "NK" else wv.shape[2]
    y = torch.full((xv.shape[0], n), float("nan"), dtype=torch.float64, device=xv.device)
    s = torch.zeros_like(y)
    at = 0
    for i, m in enumerate(splits):
        b = wv[i].t() if layout == "NK" else wv[i]
        y[at:at + m] = xv[at:at + m] @ b
        s[at:at + m] = xv[at:at + m].abs() @ b.abs()
        at += m
    return y, s


def _splits(rows, g, seed, kind="random"):
    if kind == "one":
        return [0] * (g - 1) + [rows]
    r = np.random.RandomState(seed)
    p = r.dirichlet(np.full(g, 0.4))
    s = r.multinomial(rows, p)
    if g > 2:
        s[0] += s[1]
        s[1] = 0
    return [int(v) for v in s]


GEMM_SHAPES = [  # rows, groups, N, K, layout
    (1, 1, 8, 16, "NK"), (1, 3, 256, 128, "NK"), (130, 1, 264, 144, "NK"), (129, 2, 128, 512, "NK"),
    (300, 5, 520, 640, "NK"), (1000, 7, 1000, 2064, "NK"), (777, 40, 384, 1040, "NK"),
    (600, 2, 512, 7168, "NK"), (2500, 3, 768, 1152, "NK"),
    (1, 1, 16, 16, "KN"), (1, 3, 256, 128, "KN"), (130, 1, 272, 144, "KN"), (300, 5, 528, 656, "KN"),
    (1000, 7, 1008, 2064, "KN"), (600, 2, 512, 4096, "KN"), (2500, 3, 768, 1168, "KN")]


@pytest.mark.parametrize("rows,g,n,k,layout", GEMM_SHAPES)
def test_gemm_plain(cuda_dev, rows, g, n, k, layout):
    import moe_b200
    x, w = _operands(cuda_dev, rows, g, n, k, layout, rows + n + k)
    splits = _splits(rows, g, rows + k, "one" if g == 3 and rows == 1 else "random")
    plan = moe_b200.GroupedGemmPlan(g, cuda_dev).from_splits(torch.tensor(splits))
    got = moe_b200.grouped_gemm_fp8(x, w, plan=plan, w_layout=layout).double()
    assert plan.device_error() == 0
    y, s = _product64(x, w, splits, layout)
    tol = 2.0 ** -8 * y.abs() + (1 + 2.0 ** -8) * k * 2.0 ** -24 * s
    assert bool(((got - y).abs() <= tol).all()), float(((got - y).abs() / tol.clamp_min(1e-300)).max())


def _silu64(g):
    return g / (1 + torch.exp(-g))


def _check_swiglu(rows_out, pre, y, s, k):
    f = y.shape[1] // 2
    acc = k * 2.0 ** -24 * s
    if pre is not None:
        tol = 2.0 ** -8 * y.abs() + (1 + 2.0 ** -8) * acc
        assert bool(((pre.double() - y).abs() <= tol).all())
    gate, up, eg, eu = y[:, :f], y[:, f:], acc[:, :f], acc[:, f:]
    h = _silu64(gate) * up
    # |silu'| <= 1.1; the fp32 evaluation adds a few roundings (2^-20 covers sixteen)
    eh = 1.1 * eg * (up.abs() + eu) + (_silu64(gate).abs() + 1.1 * eg) * eu + 2.0 ** -20 * h.abs() + 1e-30
    sb = ref.bytes_of(rows_out.scale)
    amax = h.abs().view(h.shape[0], -1, 128).amax(2)
    slack = eh.view(h.shape[0], -1, 128).amax(2)
    lim = 448 * torch.exp2(sb.double() - 127)
    live = amax > slack
    assert bool((amax <= lim + slack)[live].all()) and bool((2 * (amax + slack) > lim)[live].all())
    got = ref.values(rows_out.data, sb, True)
    scale = torch.exp2(sb.double() - 127).repeat_interleave(128, 1)
    tol = torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 * scale) + (1 + 2.0 ** -4) * eh
    assert bool(((got - h).abs() <= tol).all()), float(((got - h).abs() / tol).max())
    # the stored number is the rounding of a value within eh of h: away from the borders of two
    # e4m3 numbers it is the rounding of h itself
    want, _ = ref.quantize(h, True)
    same = (ref.bytes_of(rows_out.data) == ref.bytes_of(want)) | (got == 0)
    assert float(same.double().mean()) > 0.99


@pytest.mark.parametrize("rows,g,n,k", [(1, 1, 256, 16), (3, 2, 256, 144), (130, 3, 512, 512),
                                        (257, 1, 256, 1040), (900, 6, 768, 2048), (2500, 3, 512, 1152),
                                        (300, 2, 256, 7168)])
@pytest.mark.parametrize("with_pre", [False, True])
def test_gemm_swiglu(cuda_dev, rows, g, n, k, with_pre):
    import moe_b200
    x, w = _operands(cuda_dev, rows, g, n, k, "NK", rows + n, std=0.02)
    splits = _splits(rows, g, rows + n)
    plan = moe_b200.GroupedGemmPlan(g, cuda_dev).from_splits(torch.tensor(splits))
    out = moe_b200.grouped_gemm_fp8(x, w, epilogue="swiglu_fp8", plan=plan, return_pre=with_pre)
    assert plan.device_error() == 0
    q, pre = out if with_pre else (out, None)
    _check_swiglu(q, pre, *_product64(x, w, splits, "NK"), k)


@pytest.mark.parametrize("splits", [[1], [4], [5], [32], [0, 31, 1], [12, 0, 11, 3], [1] * 9 + [0] * 20])
@pytest.mark.parametrize("n,k,layout", [(256, 4112, "NK"), (264, 2048, "NK"), (2560, 1040, "NK"), (528, 4608, "KN")])
def test_gemm_few_rows(cuda_dev, splits, n, k, layout):
    """Calls of at most 32 rows share the K range of a tile between CTAs (K of 3 to 9 groups of 512)."""
    import moe_b200
    rows, g = sum(splits), len(splits)
    x, w = _operands(cuda_dev, rows, g, n, k, layout, rows + k)
    plan = moe_b200.GroupedGemmPlan(g, cuda_dev).from_splits(torch.tensor(splits))
    got = [moe_b200.grouped_gemm_fp8(x, w, plan=plan, w_layout=layout) for _ in range(3)]
    y, s = _product64(x, w, splits, layout)
    assert plan.device_error() == 0
    assert bool(((got[0].double() - y).abs() <= 2.0 ** -8 * y.abs() + 1.01 * k * 2.0 ** -24 * s).all())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    if layout == "NK" and n % 256 == 0:
        q, pre = moe_b200.grouped_gemm_fp8(x, w, plan=plan, epilogue="swiglu_fp8", return_pre=True)
        _check_swiglu(q, pre, y, s, k)


@pytest.mark.parametrize("splits", [[3, 1597], [0, 1, 128, 1919], [129, 2, 0, 1300, 17], [40, 200, 5], [255, 1, 256, 128]])
@pytest.mark.parametrize("layout", ["NK", "KN"])
def test_gemm_small_groups_beside_large(cuda_dev, splits, layout):
    """Calls of one launch (512 rows a group and more) and of two, each followed by a reader of all rows."""
    import moe_b200
    rows, k = sum(splits), 1040
    x, w = _operands(cuda_dev, rows, len(splits), 528, k, layout, 23)
    plan = moe_b200.GroupedGemmPlan(len(splits), cuda_dev).from_splits(torch.tensor(splits))
    want, s = _product64(x, w, splits, layout)
    for _ in range(20):
        again = moe_b200.grouped_gemm_fp8(x, w, plan=plan, w_layout=layout).double()  # reads behind the launches
        assert bool(((again - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * k * 2.0 ** -24 * s).all())
    assert plan.device_error() == 0


def test_gemm_rows_of_no_group_stay(cuda_dev):
    """Rows behind the last group, also inside its last tile, are not written."""
    import moe_b200
    from moe_b200 import _lib
    x, w = _operands(cuda_dev, 700, 2, 256, 256, "NK", 3)
    plan = moe_b200.GroupedGemmPlan(2, cuda_dev).from_splits(torch.tensor([300, 5]))
    out = torch.full((700, 256), 7.0, dtype=torch.bfloat16, device=cuda_dev)
    _lib.call("moe_grouped_gemm_fp8", x.data.data_ptr(), x.scale.data_ptr(), w.data.data_ptr(),
              w.scale.data_ptr(), out.data_ptr(), None, None, 700, 2, 2, 256, 256, 0, 0,
              plan.workspace.data_ptr(), plan.nbytes, torch.cuda.current_stream().cuda_stream)
    assert plan.device_error() == 0
    assert bool((out[305:] == 7.0).all())
    y, s = _product64(x, w, [300, 5], "NK")
    d = (out.double() - y)[:305].abs()
    assert bool((d <= 2.0 ** -8 * y[:305].abs() + 1.01 * 256 * 2.0 ** -24 * s[:305]).all())


def test_gemm_nonfinite_stays_in_its_row(cuda_dev):
    """A NaN in x reaches its own row, one in w its own column of its own group; nothing else."""
    import moe_b200
    for layout in ("NK", "KN"):
        rows, g, n, k = 300, 2, 272, 208  # K and N end inside a block
        gen = torch.Generator(device=cuda_dev).manual_seed(5)
        x = torch.randn(rows, k, generator=gen, device=cuda_dev)
        w = torch.randn((g, n, k) if layout == "NK" else (g, k, n), generator=gen, device=cuda_dev)
        x[7, 5] = float("inf")
        # the first reduction index of the second group, which the padded last block of the first
        # group would read if it ran past its own weight
        (w[1, 3, :1] if layout == "NK" else w[1, :1, 3]).fill_(float("nan"))
        y = moe_b200.grouped_gemm_fp8(moe_b200.quantize_fp8(x), moe_b200.quantize_fp8_weight(w),
                                      [200, 100], w_layout=layout)
        bad = torch.isnan(y)
        want = torch.zeros_like(bad)
        want[7] = True
        want[200:, 3] = True
        assert torch.equal(bad, want)


def test_gemm_scale_range(cuda_dev):
    """Far scales: products near the ends of fp32's range come out as the formula says."""
    import moe_b200
    x, w = _operands(cuda_dev, 64, 1, 128, 256, "NK", 9)
    for da, db in ((-60, -50), (60, 50), (-100, 90), (110, -120)):
        xs = (ref.bytes_of(x.scale).int() + da).clamp(0, 254).to(torch.uint8).view(torch.float8_e8m0fnu)
        ws = (ref.bytes_of(w.scale).int() + db).clamp(0, 254).to(torch.uint8).view(torch.float8_e8m0fnu)
        x2, w2 = moe_b200.Fp8Tensor(x.data, xs), moe_b200.Fp8Tensor(w.data, ws)
        got = moe_b200.grouped_gemm_fp8(x2, w2).double()
        y, s = _product64(x2, w2, [64], "NK")
        # below fp32's normal range a rounding is absolute: 2^-126 covers a flush to zero
        tol = 2.0 ** -8 * y.abs() + 1.01 * 256 * 2.0 ** -24 * s + 256 * 2.0 ** -126
        assert bool(((got - y).abs() <= tol).all())


def test_gemm_uniform_splits_streams_and_graph(cuda_dev):
    """Default splits; another stream; a captured and replayed call with new inputs."""
    import moe_b200
    x, w = _operands(cuda_dev, 100, 3, 256, 256, "NK", 11)
    base = moe_b200.grouped_gemm_fp8(x, w)
    assert torch.equal(base, moe_b200.grouped_gemm_fp8(x, w, [34, 33, 33]))
    assert torch.equal(base, moe_b200.grouped_gemm_fp8(
        x, w, torch.tensor([34, 33, 33], device=cuda_dev)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = moe_b200.grouped_gemm_fp8(x, w, [34, 33, 33])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(base, other)
    xin = torch.randn(100, 256, device=cuda_dev)
    counts = torch.tensor([34, 33, 33], dtype=torch.int32, device=cuda_dev)
    plan = moe_b200.GroupedGemmPlan(3, cuda_dev).from_splits(counts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.from_splits(counts)
        q = moe_b200.quantize_fp8(xin)
        out = moe_b200.grouped_gemm_fp8(q, w, plan=plan)
    for seed, c in ((1, [34, 33, 33]), (2, [0, 100, 0]), (3, [1, 0, 99])):
        xin.copy_(torch.randn(100, 256, generator=torch.Generator().manual_seed(seed)))
        counts.copy_(torch.tensor(c, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, moe_b200.grouped_gemm_fp8(moe_b200.quantize_fp8(xin), w, c))


def test_gemm_groups_that_share_weights(cuda_dev):
    """The group table of expert-parallel receive buffers: rows of one expert from several sources."""
    import moe_b200
    src, nw = 3, 4
    x, w = _operands(cuda_dev, 700, nw, 256, 384, "NK", 21)
    counts = [[10, 0, 200, 40], [150, 1, 129, 20], [0, 60, 50, 40]]
    plan = moe_b200.GroupedGemmPlan(src * nw, cuda_dev).from_ep_counts(
        torch.tensor(counts).flatten(), src, nw)
    got = moe_b200.grouped_gemm_fp8(x, w, plan=plan).double()
    assert plan.device_error() == 0
    at = 0
    for s in range(src):  # source-major rows
        y, m = _product64(moe_b200.Fp8Tensor(x.data[at:at + sum(counts[s])], x.scale[at:at + sum(counts[s])]),
                          w, counts[s], "NK")
        d = (got[at:at + sum(counts[s])] - y).abs()
        assert bool((d <= 2.0 ** -8 * y.abs() + 1.01 * 384 * 2.0 ** -24 * m).all())
        at += sum(counts[s])


@pytest.mark.parametrize("rows,splits", [(20, [40, 200]), (20, [5, 200]), (100, [40, 300]), (100, [300, 40]),
                                         (140, [130, 900]), (300, [10, 5000])])
def test_gemm_table_names_more_rows_than_there_are(cuda_dev, rows, splits):
    """Splits on the device are not read on the host: the rows that exist get their group's product."""
    import moe_b200
    x, w = _operands(cuda_dev, rows, 2, 512, 384, "NK", 17)
    plan = moe_b200.GroupedGemmPlan(2, cuda_dev).from_splits(torch.tensor(splits, device=cuda_dev))
    y = moe_b200.grouped_gemm_fp8(x, w, plan=plan).double()
    assert plan.device_error() == 0
    first = min(splits[0], rows)
    want, s = _product64(x, w, [first, rows - first], "NK")
    assert bool(((y - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * 384 * 2.0 ** -24 * s).all())


def test_offsets_past_32_bits(cuda_dev):
    """Outputs and inputs of more than 2^31 elements: the last rows are as those of a small call."""
    import moe_b200
    rows, n, k = 270000, 8192, 128
    x, w = _operands(cuda_dev, 4096, 2, n, k, "NK", 31)
    big = moe_b200.Fp8Tensor(x.data.repeat(66, 1)[:rows],
                             ref.bytes_of(x.scale).repeat(66, 1)[:rows].view(torch.float8_e8m0fnu))
    y = moe_b200.grouped_gemm_fp8(big, w, [100, rows - 100])
    tail = moe_b200.Fp8Tensor(big.data[-300:], big.scale[-300:])
    assert torch.equal(y[-300:], moe_b200.grouped_gemm_fp8(tail, w, [0, 300]))
    del y, big
    a = torch.randn(2048, 16384, device=cuda_dev).to(torch.bfloat16)
    q = moe_b200.quantize_fp8(a)
    qq = moe_b200.quantize_fp8(a.repeat(66, 1))
    assert torch.equal(ref.bytes_of(qq.data[-2048:]), ref.bytes_of(q.data))
    assert torch.equal(ref.bytes_of(qq.scale[-2048:]), ref.bytes_of(q.scale))
    back = moe_b200.dequantize_fp8(qq)
    assert torch.equal(back[-2048:], moe_b200.dequantize_fp8(q))

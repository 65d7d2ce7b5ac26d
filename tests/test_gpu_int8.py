"""8-bit rows and their matrix product on the GPU, against 64 bits and against the definitions in PyTorch."""
import pytest
import torch

from tensor_parallel_b200.ops import functional as OF

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _native():
    from tensor_parallel_b200.ops import native

    return native


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _wave(rows, cols, dtype, seed):
    """Activations with rows of different magnitudes and a few large channels."""
    g = _gen(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(torch.randn(rows, 1, device="cuda", generator=g))
    x[:, torch.randint(0, cols, (max(1, cols // 200),), device="cuda", generator=g)] *= 20
    return x.to(dtype)


WIDTHS = [1, 7, 8, 16, 33, 64, 250, 256, 1000, 2048, 2056, 2731, 4096, 5120, 8192, 11008, 16384, 16392, 20001, 32768, 32776, 40001]


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("cols", WIDTHS)
def test_rows(cols, dtype):
    for rows in (1, 3, 65) if cols > 256 else (1, 2, 31, 257, 4097):
        x = _wave(rows, cols, dtype, cols + rows)
        q, s = OF.quantize_int8(x)
        want = OF.quantize_int8_ref(x)
        assert torch.equal(q, want.values) and torch.equal(s, want.scales)  # two fp32 roundings each, the same ones
        assert q.stride(0) % 16 == 0 or rows == 1


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("cols", WIDTHS)
def test_rms_norm_rows(cols, with_residual, dtype):
    for rows in (1, 37):
        x = _wave(rows, cols, dtype, cols)
        res = _wave(rows, cols, dtype, cols + 1) if with_residual else None
        w = (1 + 0.1 * torch.randn(cols, device="cuda", generator=_gen(3))).to(dtype)
        for weight in (w, None):
            (q, s), h = OF.rms_norm_int8(x, weight, 1e-5, res)
            (wq, _), wh = OF.rms_norm_int8_ref(x, weight, 1e-5, res)
            assert torch.equal(q, wq) and torch.equal(h, wh)  # the integers depend on no sum
            hd = wh.double()
            v = hd if weight is None else hd * weight.double()
            scale = v.abs().amax(1).clamp_min(1e-30) / 127 * torch.rsqrt(hd.square().mean(1) + 1e-5)
            # fp32: a sum of squares (80 roundings of 2^-24 one after the other at most, halved by the root), the root, five more roundings
            torch.testing.assert_close(s.double(), scale, rtol=64 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("cols", WIDTHS)
def test_layer_norm_rows(cols, with_residual, dtype):
    rows = 37
    x = (_wave(rows, cols, dtype, cols).float() + 50).to(dtype)  # a mean that is large beside the deviation of many rows
    res = _wave(rows, cols, dtype, cols + 1) if with_residual else None
    w = (1 + 0.1 * torch.randn(cols, device="cuda", generator=_gen(3))).to(dtype)
    b = (0.1 * torch.randn(cols, device="cuda", generator=_gen(4))).to(dtype)
    for weight, bias in ((w, b), (None, None)):
        (q, s), h = OF.layer_norm_int8(x, weight, bias, 1e-5, res)
        hd = (x if res is None else (x.double() + res.double()).to(dtype)).double()
        assert torch.equal(h.double(), hd)
        y = torch.nn.functional.layer_norm(hd, (cols,), None if weight is None else weight.double(), None if bias is None else bias.double(), 1e-5)
        if cols == 1:  # (y is the bias, or zero: nothing of x is left)
            y = torch.zeros_like(y) if bias is None else bias.double().expand_as(y)
        step = y.abs().amax(1, keepdim=True).clamp_min(1e-30) / 127
        back = q.double() * s.double()[:, None]
        # half a step (and the roundings of y and of the scale, 2^-20 of 127 steps); the mean is a sum of 80 roundings of 2^-24 one after the other at
        # most, and what it is off by a small deviation magnifies (weights are below 1.5)
        slack = 80 * 2.0 ** -24 * hd.abs().amax(1, keepdim=True) * torch.rsqrt(hd.var(1, unbiased=False, keepdim=True) + 1e-5) * 1.5
        assert ((back - y).abs() <= 0.501 * step + slack).all()


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("offset,pitch", [(0, 4104), (1, 4096), (3, 4099), (8, 4112)])
def test_rows_of_other_pitches_and_alignments(offset, pitch, dtype):
    rows, cols = 19, 4080
    base = _wave(rows, pitch + 16, dtype, 5)
    x = base.as_strided((rows, cols), (pitch, 1), offset)
    q, s = OF.quantize_int8(x)
    want = OF.quantize_int8_ref(x.contiguous())
    assert torch.equal(q, want.values) and torch.equal(s, want.scales)
    wide = _wave(cols, rows, dtype, 6).t()  # columns far apart: copied
    q, s = OF.quantize_int8(wide)
    want = OF.quantize_int8_ref(wide.contiguous())
    assert torch.equal(q, want.values) and torch.equal(s, want.scales)
    res = base.as_strided((rows, cols), (pitch, 1), offset + 2)
    w = base[0].as_strided((cols,), (1,), 1)
    (q, _), h = OF.rms_norm_int8(x, w, 1e-6, res)
    (wq, _), wh = OF.rms_norm_int8_ref(x.contiguous(), w.contiguous(), 1e-6, res.contiguous())
    assert torch.equal(q, wq) and torch.equal(h, wh)


def test_leading_dimensions_and_single_rows():
    x = _wave(24, 100, BF16, 7)
    flat = OF.quantize_int8(x)
    for shape in ((2, 3, 4, 100), (1, 24, 100), (24, 1, 100)):
        q, s = OF.quantize_int8(x.view(shape))
        assert q.shape == shape and s.shape == shape[:-1] and torch.equal(q.reshape(24, 100), flat.values) and torch.equal(s.reshape(24), flat.scales)
    q, s = OF.quantize_int8(x[3])
    assert q.shape == (100,) and s.shape == () and torch.equal(q, flat.values[3])
    (q, s), h = OF.rms_norm_int8(x.view(2, 12, 100), None, 1e-6, x.view(2, 12, 100))
    assert q.shape == (2, 12, 100) and s.shape == (2, 12) and h.shape == (2, 12, 100)
    one = x[5].expand(1, 100)  # (its row stride is 0)
    assert torch.equal(OF.quantize_int8(one).values[0], flat.values[5])
    many = x[5].expand(6, 100)
    assert torch.equal(OF.quantize_int8(many).values, flat.values[5].expand(6, 100))
    assert OF.quantize_int8(x[:0]).values.shape == (0, 100)


@pytest.mark.parametrize("cols", [5, 64, 2731, 4096, 40000])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_rows_that_are_empty_or_not_finite(cols, dtype):
    x = _wave(8, cols, dtype, 8)
    x[1] = 0
    x[2, cols // 2] = float("nan")
    x[3, cols - 1] = float("inf")
    x[4, 0] = -float("inf")
    x[5] = 1e-38
    x[6] = torch.finfo(dtype).max
    for call, ref in ((OF.quantize_int8, OF.quantize_int8_ref),
                      (lambda t: OF.rms_norm_int8(t, None, 1e-6)[0], lambda t: OF.rms_norm_int8_ref(t, None, 1e-6)[0])):
        (q, s), want = call(x), ref(x)
        assert torch.equal(q, want.values)
        assert torch.isnan(s[2:5]).all() and not q[2:5].any() and not q[1].any()
        torch.testing.assert_close(s, want.scales, rtol=1e-5, atol=0, equal_nan=True)
    q, s = OF.layer_norm_int8(x, None, None)[0]
    assert torch.isnan(s[2:5]).all() and not q[2:5].any() and torch.isfinite(s[:2]).all()


def test_only_the_rows_are_written():
    nat = _native()
    for cols in (64, 100, 4096, 4100):
        x = _wave(5, cols, BF16, 9)
        pitch = (cols + 15) // 16 * 16 + 16
        room = torch.full((9, pitch), 77, dtype=torch.int8, device="cuda")
        scales = torch.full((9,), 5.0, device="cuda")
        nat.rows_int8(x, out=OF.Int8Rows(room[2:7, :cols], scales[2:7]))
        assert (room[:2] == 77).all() and (room[7:] == 77).all() and (room[:, cols:] == 77).all()
        assert (scales[:2] == 5).all() and (scales[7:] == 5).all()
        assert torch.equal(room[2:7, :cols], OF.quantize_int8_ref(x).values)


def test_the_sum_in_place_of_x():
    nat = _native()
    for cols in (96, 101, 4096, 40000):
        x, r = _wave(6, cols, BF16, 10), _wave(6, cols, BF16, 11)
        (wq, ws), wh = OF.rms_norm_int8_ref(x, None, 1e-6, r)
        q, s = nat.rows_int8(x, eps=1e-6, norm=0, residual=r, sum_out=x)
        assert torch.equal(q, wq) and torch.equal(x, wh)


def _operands(tokens, features, k, seed):
    x = OF.quantize_int8_ref(_wave(tokens, k, torch.float32, seed))
    w = OF.quantize_int8_ref(torch.randn(features, k, device="cuda", generator=_gen(seed + 1)) / k ** 0.5)
    return x, w


def _act64(v, act):
    if act == "swiglu16":
        g = v.unflatten(-1, (-1, 2, 16))
        return (torch.nn.functional.silu(g[..., 0, :]) * g[..., 1, :]).flatten(-2)
    return {None: lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
            "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[act](v)


def _check_product(x, w, bias=None, act=None, residual=None):
    before = _native().launch_count
    out = OF.linear_int8(x, w, bias, act, residual)
    assert _native().launch_count > before
    sums = (x.values.double() @ w.values.double().t())
    v = sums * x.scales.double()[..., None] * w.scales.double()
    size = v.abs()
    if bias is not None:
        v, size = v + bias.double(), size + bias.double().abs()
    want = _act64(v, act)
    # fp32 in front of the activation: four roundings of 2^-24 of the terms; the activations' slopes stay below 1.2, a gated pair's below the other half
    slack = 8 * 2.0 ** -24 * size * 1.2
    if act == "swiglu16":
        (g, u), (sg, su) = (t.unflatten(-1, (-1, 2, 16)).unbind(-2) for t in (v, slack))
        slack = (sg * u.abs() + su * g.abs()).flatten(-2) + 2.0 ** -20 * want.abs()
    if residual is not None:
        want = want + residual.double()
    # one rounding to bf16 (2^-8 of the result at most), what lies below 1e-30 is of no account, and the activations' own functions (a few 2^-22 of a value of size 1)
    bound = 2.0 ** -8 * want.abs() * 1.001 + slack + (2.0 ** -20 * (1 + size if act != "swiglu16" else want.abs()) if act else 0) + 1e-30
    assert out.dtype == BF16 and out.shape == want.shape
    assert ((out.double() - want).abs() <= bound).all(), (out.double() - want).abs().max()
    return out


TOKENS = [1, 2, 8, 9, 16, 17, 33, 64, 65, 100, 128, 129, 200, 256, 257, 300, 511, 513, 1000]


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("features,k", [(1, 1), (5, 16), (33, 100), (64, 64), (128, 1001), (1000, 520), (4096, 4096), (4737, 257), (9600, 130)])
def test_product_sizes(tokens, features, k):
    x, w = _operands(tokens, features, k, tokens + features)
    _check_product(x, w)


@pytest.mark.parametrize("tokens", [1, 8, 40, 64, 100, 300, 700])
@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu", "swiglu16"])
@pytest.mark.parametrize("features,k", [(2048, 512), (4800, 1000), (32, 2048), (999, 333)])
def test_product_epilogues(tokens, features, k, act):
    if act == "swiglu16":
        features = (features + 31) // 32 * 32
    x, w = _operands(tokens, features, k, 20)
    bias = torch.randn(features, device="cuda", generator=_gen(21)).to(BF16)
    residual = None if act == "swiglu16" else torch.randn(tokens, features, device="cuda", generator=_gen(22)).to(BF16)
    _check_product(x, w, bias, act, residual)
    _check_product(x, w, None, act, residual)
    _check_product(x, w, bias, act, None)


@pytest.mark.parametrize("tokens", [1, 16, 64, 130, 520])
@pytest.mark.parametrize("k", [64, 4096, 11008, 131071])
def test_sums_are_exact_integers(tokens, k):
    """Sums of extreme integers: only exact 32-bit arithmetic gives these, up to the ends of the range."""
    x = torch.full((tokens, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((96, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    w[2, 1::2] = 127
    w[3] = 0
    w[3, k - 1] = 1
    x, w = OF.Int8Rows(_native()._int8_ready(x), torch.full((tokens,), 2.0 ** -10, device="cuda")), OF.Int8Rows(_native()._int8_ready(w), torch.ones(96, device="cuda"))
    out = OF.linear_int8(x, w)
    want = (x.values.double() @ w.values.double().t()) * 2.0 ** -10
    assert torch.equal(out, want.float().to(BF16))


def test_product_does_not_read_between_the_rows_and_writes_only_its_result():
    nat = _native()
    for tokens, features, k in ((7, 70, 100), (90, 300, 200), (300, 260, 72)):
        x, w = _operands(tokens, features, k, 30)
        pitch = (k + 15) // 16 * 16 + 32
        xp, wp = (torch.full((n, pitch), 113, dtype=torch.int8, device="cuda") for n in (tokens + 4, features + 4))
        xp[2:tokens + 2, :k], wp[2:features + 2, :k] = x.values, w.values
        room = torch.full((tokens + 4, features + 9), 3.0, dtype=BF16, device="cuda")
        out = nat.gemm_int8(OF.Int8Rows(xp[2:tokens + 2, :k], x.scales), OF.Int8Rows(wp[2:features + 2, :k], w.scales), out=room[2:tokens + 2, 4:features + 4])
        assert torch.equal(out, _check_product(x, w))
        assert (room[:2] == 3).all() and (room[tokens + 2:] == 3).all() and (room[:, :4] == 3).all() and (room[:, features + 4:] == 3).all()


@pytest.mark.parametrize("tokens", [3, 100, 600])
def test_product_of_unaligned_operands_and_residual_in_place(tokens):
    nat = _native()
    features, k = 300, 130
    x, w = _operands(tokens, features, k, 40)
    want = _check_product(x, w)
    for ld in (k, k + 1):  # rows that no tensor map can describe
        xu = torch.empty(tokens * ld + 3, dtype=torch.int8, device="cuda")[3:].as_strided((tokens, k), (ld, 1))
        wu = torch.empty(features * ld + 1, dtype=torch.int8, device="cuda")[1:].as_strided((features, k), (ld, 1))
        xu.copy_(x.values)
        wu.copy_(w.values)
        assert torch.equal(OF.linear_int8(OF.Int8Rows(xu, x.scales), OF.Int8Rows(wu, w.scales)), want)
    cols = OF.Int8Rows(w.values.t().contiguous().t(), w.scales)  # a weight that lies transposed
    assert torch.equal(OF.linear_int8(x, cols), want)
    r = torch.randn(tokens, features, device="cuda", generator=_gen(41)).to(BF16)
    out = _check_product(x, w, residual=r)
    again = nat.gemm_int8(x, w, residual=r, out=r)
    assert again is r and torch.equal(r, out)


@pytest.mark.parametrize("tokens", [2, 80, 400])
def test_rows_that_are_not_finite_stay_so(tokens):
    x, w = _operands(tokens, 256, 128, 50)
    want = OF.linear_int8(x, w)
    scales = x.scales.clone()
    scales[1] = float("nan")
    ws = w.scales.clone()
    ws[7] = float("inf")
    out = OF.linear_int8(OF.Int8Rows(x.values, scales), OF.Int8Rows(w.values, ws))
    assert torch.isnan(out[1]).all() and not torch.isfinite(out[:, 7]).any()
    keep = torch.ones(tokens, dtype=torch.bool, device="cuda")
    keep[1] = False
    cols = torch.arange(256, device="cuda") != 7
    assert torch.equal(out[keep][:, cols], want[keep][:, cols])


def test_result_does_not_depend_on_the_other_tokens():
    x, w = _operands(700, 512, 768, 60)
    whole = OF.linear_int8(x, w)
    for n in (1, 16, 33, 64, 65, 128, 300, 600):
        assert torch.equal(OF.linear_int8(OF.Int8Rows(x.values[:n], x.scales[:n]), w), whole[:n])


def test_calls_in_flight_on_two_streams_and_in_replayed_graphs():
    x, w = _operands(64, 4096, 2048, 70)
    y = _wave(64, 2048, BF16, 71)
    gamma = torch.ones(2048, device="cuda", dtype=BF16)

    def run():
        rows, h = OF.rms_norm_int8(y, gamma, 1e-5, y)
        return OF.linear_int8(rows, w), OF.linear_int8(x, w), OF.quantize_int8(h)

    def flat(t):
        return [t[0], t[1], *t[2]]

    want = flat(run())
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(flat(run()))
    torch.cuda.synchronize()
    graphs, results = [], []
    for s in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            results.append(flat(run()))
        graphs.append(g)
    for _ in range(3):
        for g, s in zip(graphs, streams):  # two graphs at once: no workspace that they could share
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for r in got + results:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    _native().device_state(torch.device("cuda", torch.cuda.current_device())).check_status()


def test_refusals_on_the_gpu():
    x, w = _operands(4, 64, 64, 80)
    with pytest.raises(ValueError):
        OF.linear_int8(x, OF.Int8Rows(w.values.cpu(), w.scales.cpu()))
    with pytest.raises(ValueError):
        OF.linear_int8(x, OF.Int8Rows(w.values, w.scales.cpu()))
    with pytest.raises(ValueError):
        OF.linear_int8(x, w, torch.zeros(64, dtype=BF16))
    with pytest.raises(ValueError):
        OF.rms_norm_int8(torch.randn(2, 8, device="cuda"), torch.ones(8))
    with pytest.raises(TypeError):
        OF.quantize_int8(torch.randn(2, 8, device="cuda").half())
    with pytest.raises(RuntimeError, match="no gradient"):
        OF.quantize_int8(torch.randn(2, 8, device="cuda", requires_grad=True))
    nat = _native()
    # the entry points' own checks: nothing is launched
    status = nat._ptr(nat.device_state(torch.device("cuda", 0)).status)

    def entry(**kw):
        a = dict(x=nat._ptr(x.values), w=nat._ptr(w.values), tokens=4, features=64, k=64, ldx=64, ldw=64, ld_out=64, act=0, residual=None)
        a.update(kw)
        out = torch.zeros(4, 64, device="cuda", dtype=BF16)
        code = nat.LIB.tpb_gemm_int8(a["x"], nat._ptr(x.scales), a["w"], nat._ptr(w.scales), nat._ptr(out), None, a["residual"], a["tokens"], a["features"], a["k"],
                                     a["ldx"], a["ldw"], a["ld_out"], 0, a["act"], 0, status, nat._stream())
        torch.cuda.synchronize()
        return code

    assert entry() == 0
    assert entry(x=nat._ptr(x.values) + 1) == 2 and entry(ldw=72) == 2
    assert entry(ldx=48) == 1 and entry(ld_out=63) == 1 and entry(tokens=0) == 1 and entry(act=6) == 1 and entry(x=None) == 1
    assert entry(act=5, residual=status) == 1 and entry(act=5, features=48) == 1
    assert entry(k=131072, ldx=131072, ldw=131072) == 7


def test_a_gated_mlp_in_8_bits():
    """The run of operators that a decoder layer's MLP is: norm with the residual's addition, gate and up, rows of the activation, down with the residual."""
    nat = _native()
    tokens, hidden, ffn = 37, 512, 1376
    g = _gen(90)
    x, r = _wave(tokens, hidden, BF16, 91), _wave(tokens, hidden, BF16, 92)
    gamma = (1 + 0.1 * torch.randn(hidden, device="cuda", generator=g)).to(BF16)
    wg, wu = (torch.randn(ffn, hidden, device="cuda", generator=g).to(BF16) / hidden ** 0.5 for _ in range(2))
    wd = torch.randn(hidden, ffn, device="cuda", generator=g).to(BF16) / ffn ** 0.5
    w1, w2 = OF.quantize_int8(nat.interleave_gate_up(wg, wu)), OF.quantize_int8(wd)
    rows, h = OF.rms_norm_int8(x, gamma, 1e-5, r)
    act = OF.linear_int8(rows, w1, act="swiglu16")
    mid = OF.quantize_int8(act)
    out = OF.linear_int8(mid, w2, residual=h)
    # each step against its definition on the same inputs
    (wr, ws), wh = OF.rms_norm_int8_ref(x, gamma, 1e-5, r)
    assert torch.equal(rows.values, wr) and torch.equal(h, wh)
    v = rows.dequantize(torch.float64) @ w1.dequantize(torch.float64).t()
    want = _act64(v, "swiglu16")
    assert ((act.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * v.abs().max() ** 2).all()
    assert torch.equal(mid.values, OF.quantize_int8_ref(act).values)
    want = mid.dequantize(torch.float64) @ w2.dequantize(torch.float64).t() + h.double()
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * want.abs().max()).all()
    # and the whole near the layer it stands for.  A step is 1/127 of a row's largest value, 60 deviations with the large channels here, so that a
    # row's error (a step / sqrt(12)) is about 0.14 deviations, 0.09 of its root mean square; gate and up both carry it, the activation its own
    n = OF.rms_norm_ref(h, gamma, 1e-5).double()
    exact = (torch.nn.functional.silu(n @ wg.double().t()) * (n @ wu.double().t())) @ wd.double().t() + h.double()
    assert (out.double() - exact).norm() < 0.25 * (exact - h.double()).norm()


def test_offsets_beyond_32_bits():
    rows, cols = 70001, 32768  # 2.3 G elements
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    some = torch.tensor([0, 1, 65535, 65536, 65537, 69999, 70000], device="cuda")
    x[some] = _wave(len(some), cols, BF16, 100)
    q, s = OF.quantize_int8(x)
    want = OF.quantize_int8_ref(x[some])
    assert torch.equal(q[some], want.values) and torch.equal(s[some], want.scales)
    assert not q[2:65535:4099].any()
    (nq, ns), h = OF.rms_norm_int8(x, None, 1e-6, x)
    (wq, ws), wh = OF.rms_norm_int8_ref(x[some], None, 1e-6, x[some])
    assert torch.equal(nq[some], wq) and torch.equal(h[some], wh)
    torch.testing.assert_close(ns[some], ws, rtol=64 * 2.0 ** -24, atol=0)
    del h, nq, ns
    w = OF.quantize_int8_ref(torch.randn(40, cols, device="cuda", generator=_gen(101)))
    out = OF.linear_int8(OF.Int8Rows(q, s), w)
    assert torch.equal(out[some], OF.linear_int8(OF.Int8Rows(q[some].contiguous(), s[some]), w)) and not out[2:65535:4099].any()
    del q, s, x, out
    tokens, features, k = 131077, 20000, 64  # 2.6 G results
    x, w = _operands(tokens, features, k, 102)
    out = OF.linear_int8(x, w)
    some = torch.tensor([0, 127, 107373, 107374, 107375, 131071, 131072, 131076], device="cuda")
    assert torch.equal(out[some], OF.linear_int8(OF.Int8Rows(x.values[some].contiguous(), x.scales[some]), w))


def test_strided_leading_dimensions():
    x = _wave(40, 96, BF16, 110).view(4, 10, 96)
    for t in (x[:, ::2], x.transpose(0, 1), x[::2], x[:, 3:4], x[1:2, :, :], x[..., 16:80], x[..., 5:70]):
        got, want = OF.quantize_int8(t), OF.quantize_int8_ref(t)
        assert got.values.shape == t.shape and torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales)
        (q, s), h = OF.rms_norm_int8(t, None, 1e-6, t)
        assert torch.equal(h, (t.float() * 2).to(BF16)) and torch.equal(q, want.values)
    w = OF.quantize_int8(_wave(64, 96, BF16, 111))
    r = OF.quantize_int8(x)
    for at in ((slice(None), slice(None, None, 2)), (slice(1, 3),), (slice(None), slice(4, 5))):
        part = OF.Int8Rows(r.values[at], r.scales[at])
        residual = _wave(part.scales.numel(), 64, BF16, 112).view(*part.scales.shape, 64)
        assert torch.equal(OF.linear_int8(part, w), OF.linear_int8(r, w)[at])
        want = OF.linear_int8_ref(part, w, residual=residual).float()
        torch.testing.assert_close(OF.linear_int8(part, w, residual=residual).float(), want, rtol=2.0 ** -7, atol=1e-4)  # a rounding to bf16 on either side


def test_under_transforms_tracing_and_tangents():
    x = _wave(6, 64, BF16, 120)
    want = OF.quantize_int8_ref(x)
    got = torch.vmap(lambda t: tuple(OF.quantize_int8(t)))(x.view(2, 3, 64))
    assert torch.equal(got[0].reshape(6, 64), want.values) and torch.equal(got[1].reshape(6), want.scales)
    traced = torch.jit.trace(lambda t: tuple(OF.quantize_int8(t)), (x,))
    y = _wave(6, 64, BF16, 121)
    assert torch.equal(traced(y)[0], OF.quantize_int8_ref(y).values)  # (its steps, not its first result)
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no derivative"):
            OF.quantize_int8(dual)
        with pytest.raises(RuntimeError, match="no derivative"):
            OF.rms_norm_int8(x, None, 1e-6, residual=dual)
    with torch.inference_mode():
        got = OF.quantize_int8(x)
        assert torch.equal(got.values, want.values) and got.values.is_inference()
        got.values.zero_()


def test_a_weight_of_another_type_and_rows_as_a_plain_pair():
    x = _wave(5, 64, BF16, 130)
    w = 1 + 0.1 * torch.randn(64, device="cuda", generator=_gen(131))
    (q, s), _ = OF.rms_norm_int8(x, w, 1e-6)
    (wq, ws), _ = OF.rms_norm_int8_ref(x, w, 1e-6)
    assert torch.equal(q, wq)
    rows, weight = OF.quantize_int8(x), OF.quantize_int8(_wave(32, 64, BF16, 132))
    assert torch.equal(OF.linear_int8(tuple(rows), tuple(weight)), OF.linear_int8(rows, weight))


@pytest.mark.multigpu
def test_tensors_on_another_device_than_the_current_one():
    x, w = _operands(9, 64, 128, 140)
    y = _wave(9, 128, BF16, 141)
    want, rows = OF.linear_int8(x, w), OF.quantize_int8(y)
    with torch.cuda.device(0):
        far = [OF.Int8Rows(t.values.to("cuda:1"), t.scales.to("cuda:1")) for t in (x, w)]
        out, got = OF.linear_int8(*far), OF.quantize_int8(y.to("cuda:1"))
    assert out.device.index == 1 and torch.equal(out.cpu(), want.cpu()) and torch.equal(got.values.cpu(), rows.values.cpu())


@pytest.mark.parametrize("shape", [(5, 40), (2, 3, 64), (33,)])
def test_rows_are_saved_and_copied_like_other_tensors(shape, tmp_path):
    import copy

    rows = OF.quantize_int8(_wave(1, torch.Size(shape).numel(), BF16, 95).view(shape))
    torch.save({"weight": rows.values, "scales": rows.scales}, tmp_path / "rows.pt")
    read = torch.load(tmp_path / "rows.pt", weights_only=True)
    assert torch.equal(read["weight"], rows.values) and torch.equal(read["scales"], rows.scales)
    twin = copy.deepcopy(rows)
    twin.values.zero_()
    twin.scales.zero_()
    again = OF.quantize_int8(_wave(1, torch.Size(shape).numel(), BF16, 95).view(shape))
    assert torch.equal(again.values, rows.values) and torch.equal(again.scales, rows.scales)


# Rows of these widths and numbers (in SMs) reach every division of a row among threads, and the kernel that has rows on their way ahead.
MANY = [(3584, 5), (4096, 5), (4100, 3), (4104, 17), (5120, 5), (6152, 3), (8192, 17), (8196, 3), (8200, 5), (11008, 3), (11008, 17), (16384, 13), (16392, 5), (20000, 2), (32768, 3), (32776, 3)]


def _many(cols, sms, dtype, seed):
    rows = sms * torch.cuda.get_device_properties(0).multi_processor_count + 3
    x = _wave(rows, cols, dtype, seed)
    x[1] = 0
    x[2, cols - 1] = float("nan")
    return x


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("cols,sms", MANY)
def test_many_wide_rows(cols, sms, dtype):
    x = _many(cols, sms, dtype, cols)
    q, s = OF.quantize_int8(x)
    want = OF.quantize_int8_ref(x)
    assert torch.equal(q, want.values)
    torch.testing.assert_close(s, want.scales, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("cols,sms", MANY)
def test_rms_norm_of_many_wide_rows(cols, sms, with_residual, dtype):
    x = _many(cols, sms, dtype, cols)
    res = _wave(*x.shape, dtype, cols + 1) if with_residual else None
    w = (1 + 0.1 * torch.randn(cols, device="cuda", generator=_gen(3))).to(dtype)
    (q, s), h = OF.rms_norm_int8(x, w, 1e-5, res)
    (wq, ws), wh = OF.rms_norm_int8_ref(x, w, 1e-5, res)
    assert torch.equal(q, wq)
    torch.testing.assert_close(h, wh, rtol=0, atol=0, equal_nan=True)
    most = (wh.float() * w.float()).abs().amax(1).clamp_min(1e-30)
    scale = most.double() / 127 * torch.rsqrt((wh.float() * wh.float()).sum(1, dtype=torch.float64) / cols + 1e-5)
    # fp32: a square, then at most 80 sums one after the other (halved by the root), the root, five more roundings, and the squares' above
    torch.testing.assert_close(s.double(), scale, rtol=64 * 2.0 ** -24, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("cols,sms", MANY)
def test_layer_norm_of_many_wide_rows(cols, sms, with_residual, dtype):
    x = (_many(cols, sms, dtype, cols).float() + 50).to(dtype)
    res = _wave(*x.shape, dtype, cols + 1) if with_residual else None
    w = (1 + 0.1 * torch.randn(cols, device="cuda", generator=_gen(3))).to(dtype)
    b = (0.1 * torch.randn(cols, device="cuda", generator=_gen(4))).to(dtype)
    (q, s), h = OF.layer_norm_int8(x, w, b, 1e-5, res)
    torch.testing.assert_close(h, x if res is None else (x.float() + res.float()).to(dtype), rtol=0, atol=0, equal_nan=True)
    assert s[2].isnan() and not q[2].any()
    for lo in range(0, x.shape[0], 512):
        part = slice(lo, lo + 512)
        hd = h[part].double()
        y = torch.nn.functional.layer_norm(hd, (cols,), w.double(), b.double(), 1e-5)
        step = y.abs().amax(1, keepdim=True).clamp_min(1e-30) / 127
        back = q[part].double() * s[part].double()[:, None]
        slack = 80 * 2.0 ** -24 * hd.abs().amax(1, keepdim=True) * torch.rsqrt(hd.var(1, unbiased=False, keepdim=True) + 1e-5) * 1.5
        near = (back - y).abs() <= 0.501 * step + slack  # (as in test_layer_norm_rows)
        assert (near | ~hd.isfinite().all(1, keepdim=True)).all()


# tokens, features that the widths of the pair kernel's tile take on a GPU of 148 SMs
PAIRS = {128: [(512, 4096), (500, 4095)], 160: [(300, 11008), (290, 11009)], 192: [(300, 12288), (511, 12285)], 224: [(300, 22016), (2048, 12288)], 256: [(768, 12288), (1000, 4090)]}


@pytest.mark.parametrize("act", [None, "gelu", "swiglu16"])
@pytest.mark.parametrize("width", list(PAIRS))
def test_every_width_of_the_pair_tile(width, act):
    import ctypes

    for tokens, features in PAIRS[width]:
        features = features // 32 * 32 if act == "swiglu16" else features
        k = 4112 if features % 8 else 400  # (unaligned results of a short contraction go to another kernel)
        form = (ctypes.c_int * 2)()
        if torch.cuda.get_device_properties(0).multi_processor_count == 148:
            assert _native().LIB.tpb_gemm_int8_form(tokens, features, k, 148, form) == 2 and form[0] == width, (tokens, features, form[0])
        x, w = _operands(tokens, features, k, width + tokens)
        bias = torch.randn(features, device="cuda", generator=_gen(5)).to(BF16)
        residual = None if act else torch.randn(tokens, features, device="cuda", generator=_gen(6)).to(BF16)
        _check_product(x, w, bias, act, residual)


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("cols,sms", [(768, 33), (1000, 33), (1024, 40), (1032, 17), (1536, 17), (2048, 70), (2056, 17), (3584, 17), (3592, 17), (4096, 40), (4104, 17), (8192, 17), (8200, 17), (16384, 17)])
def test_norms_without_a_residual_of_many_rows(cols, sms, weighted):
    rows = sms * torch.cuda.get_device_properties(0).multi_processor_count + 1
    pitch = cols + 24
    x = _wave(rows, pitch, BF16, cols).as_strided((rows, cols), (pitch, 1), 8)
    x[1], x[rows - 1, 0], x[2, cols - 1] = 0, float("inf"), float("nan")
    w, b = ((1 + 0.1 * torch.randn(cols, device="cuda", generator=_gen(3))).to(BF16), (0.1 * torch.randn(cols, device="cuda", generator=_gen(4))).to(BF16)) if weighted else (None, None)
    (q, s), _ = OF.rms_norm_int8(x, w, 1e-5)
    v = x.float() if w is None else x.float() * w.float()
    want = OF.rms_norm_int8_ref(x, w, 1e-5)[0]
    assert torch.equal(q, want.values)
    scale = v.abs().amax(1).clamp_min(1e-30).double() / 127 * torch.rsqrt((x.float() * x.float()).sum(1, dtype=torch.float64) / cols + 1e-5)
    finite = scale.isfinite()
    assert finite.sum() == rows - 2 and s[~finite].isnan().all() and not q[~finite].any()
    torch.testing.assert_close(s[finite].double(), scale[finite], rtol=64 * 2.0 ** -24, atol=0)  # (as in test_rms_norm_of_many_wide_rows)
    (q, s), _ = OF.layer_norm_int8(x, w, b, 1e-5)
    assert s[~finite].isnan().all() and not q[~finite].any()
    xd = x[finite].double()
    y = torch.nn.functional.layer_norm(xd, (cols,), None if w is None else w.double(), None if b is None else b.double(), 1e-5)
    step = y.abs().amax(1, keepdim=True).clamp_min(1e-30) / 127
    back = q[finite].double() * s[finite].double()[:, None]
    slack = 80 * 2.0 ** -24 * xd.abs().amax(1, keepdim=True) * torch.rsqrt(xd.var(1, unbiased=False, keepdim=True) + 1e-5) * 1.5
    assert ((back - y).abs() <= 0.501 * step + slack).all()  # (as in test_layer_norm_rows)


@pytest.mark.parametrize("cols,sms", [(1024, 33), (2048, 5), (4096, 5), (8192, 5), (11008, 5), (4096, 40), (20000, 3)])
def test_the_sum_of_many_rows_in_place(cols, sms):
    nat = _native()
    x = _many(cols, sms, BF16, cols)
    res = _wave(*x.shape, BF16, cols + 1)
    for norm, ref in ((0, lambda: OF.rms_norm_int8_ref(x, None, 1e-5, res)), (1, lambda: OF.layer_norm_int8(x, None, None, 1e-5, res))):
        (wq, _), wh = ref()
        for target in ("x", "residual"):
            a, b = x.clone(), res.clone()
            into = a if target == "x" else b
            q, _ = nat.rows_int8(a, eps=1e-5, norm=norm, residual=b, sum_out=into)
            assert torch.equal(q, wq)
            torch.testing.assert_close(into, wh, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("act,residual", [(None, True), ("gelu", False), ("silu", True)])
@pytest.mark.parametrize("tokens,features,k", [(150, 6370, 512), (300, 12345, 500), (1000, 1565, 2048), (1300, 3043, 130)])
def test_unaligned_results_of_short_contractions(tokens, features, k, act, residual):
    x, w = _operands(tokens, features, k, tokens)
    bias = torch.randn(features, device="cuda", generator=_gen(5)).to(BF16)
    out = _check_product(x, w, bias, act, torch.randn(tokens, features, device="cuda", generator=_gen(6)).to(BF16) if residual else None)
    if not residual:  # the same results in rows that are aligned: by another kernel, bit by bit
        room = torch.zeros(tokens, (features + 31) // 32 * 32, device="cuda", dtype=BF16)
        assert torch.equal(_native().gemm_int8(x, w, bias, act, out=room[:, :features]), out) and not room[:, features:].any()


@pytest.mark.parametrize("cols,sms", [(4490, 5), (5255, 5), (8191, 3), (8191, 9), (11007, 3), (11007, 9), (16383, 9), (16610, 1), (32767, 1)])
def test_many_rows_of_odd_widths(cols, sms):
    test_many_wide_rows(cols, sms, BF16)
    for with_residual in (False, True):
        test_rms_norm_of_many_wide_rows(cols, sms, with_residual, BF16)
        test_layer_norm_of_many_wide_rows(cols, sms, with_residual, BF16)

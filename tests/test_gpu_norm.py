"""RMS norm with the residual's addition and its 8-bit output blocks, and the products that read them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


@pytest.fixture(scope="module")
def dev(cuda_lib):
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def inputs(seed, m, k, dtype, w_dtype=None, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(m, k, generator=g) * scale).to(dtype)
    r = (torch.randn(m, k, generator=g) * 3).to(dtype)
    w = (1 + 0.2 * torch.randn(k, generator=g)).to(w_dtype or dtype)
    return x, r, w


def steps(x, r, w, eps=EPS):
    """h as stored and the f32 values of y, every rounding of the definition in its place (numpy)."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    hf, wf = h.float().numpy(), w.float().numpy()
    with np.errstate(all="ignore"):
        inv = (1.0 / np.sqrt((hf.astype(np.float64) ** 2).sum(-1, keepdims=True) / hf.shape[-1] + eps)).astype(np.float32)
        return h, (hf * inv) * wf


def check_values(y, x, r, w):
    """y against the formula in 64 bits: three roundings to f32 (inv, h * inv, the product) and one to the type."""
    h, _ = steps(x, r, w)
    hd, wd = h.double(), w.double()
    want = hd / ((hd ** 2).mean(-1, keepdim=True) + EPS).sqrt() * wd
    u = 0.0 if y.dtype == torch.float32 else torch.finfo(y.dtype).eps / 2
    tol = want.abs() * ((1 + 2.0 ** -24) ** 3 * (1 + u) * (1 + 1e-12) - 1) + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    assert ((y.cpu().double() - want).abs() <= tol).all()


SHAPES = [(1, 1), (1, 7), (3, 8), (9, 33), (5, 256), (2, 264), (7, 1000), (1, 4096), (4, 4099), (2, 8192), (1, 20000), (2, 40000), (3, 33001), (300, 128)]


@pytest.mark.parametrize("x", TYPES)
@pytest.mark.parametrize("m,k", SHAPES)
def test_values(dev, m, k, x):
    from lloom_b200 import rms_norm

    for w_type in ("f32", x):
        for residual in (False, True):
            a, r, w = inputs(m * k, m, k, TYPES[x], TYPES[w_type])
            r = r if residual else None
            got = rms_norm(a.to(dev), w.to(dev), EPS, None if r is None else r.to(dev))
            y, h = got if residual else (got, None)
            assert y.shape == a.shape and y.dtype == a.dtype
            check_values(y, a, r, w)
            if residual:
                assert torch.equal(h.cpu(), steps(a, r, w)[0])


@pytest.mark.parametrize("fmt", ["Q4_0", "Q5_0", "Q8_0", "Q4K", "Q5K", "Q6K"])
@pytest.mark.parametrize("x", TYPES)
@pytest.mark.parametrize("m,blocks", [(1, 1), (3, 2), (1, 16), (5, 9), (2, 40), (1, 130), (2, 160)])
def test_blocks(dev, oracle, fmt, x, m, blocks):
    """The blocks are the reference quantizer's on the f32 values, byte for byte."""
    from lloom_b200 import GgmlDType, QActs, rms_norm
    from lloom_b200.quantized import act_type

    dt = getattr(GgmlDType, fmt)
    k = blocks * 256 if fmt.endswith("K") else blocks * 256 - 32 * (blocks % 3)
    a, r, w = inputs(blocks, m, k, TYPES[x])
    for res in (None, r):
        got = rms_norm(a.to(dev), w.to(dev), EPS, None if res is None else res.to(dev), act_for=dt)
        acts = got if res is None else got[0]
        assert isinstance(acts, QActs) and acts.dtype == act_type(dt) and acts.shape == (m, k)
        _, y = steps(a, res, w)
        want = oracle.quantize_act(int(dt), y)
        np.testing.assert_array_equal(acts.blocks.cpu().numpy(), want)
        # and what they stand for
        if acts.dtype == GgmlDType.Q8_0:
            blk = want.reshape(-1, 34)
            val = blk[:, :2].copy().view(np.float16).astype(np.float32) * blk[:, 2:].view(np.int8).astype(np.float32)
        else:
            blk = want.reshape(-1, 292)
            val = blk[:, :4].copy().view(np.float32) * blk[:, 4:260].copy().view(np.int8).astype(np.float32)
        np.testing.assert_array_equal(acts.dequantize().cpu().numpy(), val.reshape(m, k))


def test_rows_apart_and_off_the_boundary(dev):
    """Strided rows, a base that is off 16 bytes, and a three-dimensional stream give the contiguous call's bits."""
    from lloom_b200 import GgmlDType, rms_norm

    a, r, w = inputs(5, 6, 512, torch.float32)
    wide = torch.zeros(6, 1200, device=dev)
    wide[:, 3:515] = a.to(dev)
    rd, wd = r.to(dev), w.to(dev)
    off = torch.zeros(513, device=dev)
    off[1:] = wd
    want = rms_norm(a.to(dev), wd, EPS, rd)
    want_q = rms_norm(a.to(dev), wd, EPS, rd, act_for=GgmlDType.Q6K)
    for xs, ws in ((wide[:, 3:515], wd), (wide[:, 3:515], off[1:]), (a.to(dev), off[1:])):
        got = rms_norm(xs, ws, EPS, rd)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(rms_norm(xs, ws, EPS, rd, act_for=GgmlDType.Q6K)[0].blocks, want_q[0].blocks)
    three = rms_norm(a.to(dev).view(2, 3, 512), wd, EPS, rd.view(2, 3, 512))
    assert three[0].shape == (2, 3, 512) and torch.equal(three[0].view(6, 512), want[0])
    one = rms_norm(a[0].to(dev), wd)
    assert one.shape == (512,)


def test_a_row_does_not_depend_on_the_batch(dev):
    from lloom_b200 import GgmlDType, rms_norm

    a, r, w = (t.to(dev) for t in inputs(6, 2000, 2048, torch.bfloat16))
    y, h = rms_norm(a, w, EPS, r)
    q, _ = rms_norm(a, w, EPS, r, act_for=GgmlDType.Q8_0)
    for i in (0, 999, 1999):
        yi, hi = rms_norm(a[i:i + 1], w, EPS, r[i:i + 1])
        qi, _ = rms_norm(a[i:i + 1], w, EPS, r[i:i + 1], act_for=GgmlDType.Q8_0)
        assert torch.equal(yi[0], y[i]) and torch.equal(hi[0], h[i]) and torch.equal(qi.blocks[0], q.blocks[i])


def test_extreme_rows(dev, oracle):
    """A zero row, tiny and huge rows (their squares leave the range of 32 bits), a NaN and an infinity: as the formula has them."""
    from lloom_b200 import GgmlDType, rms_norm

    a = torch.randn(7, 512, generator=torch.Generator().manual_seed(1))
    a[0] = 0
    a[1] *= 1e-30
    a[2] *= 1e30
    a[3, 5] = float("nan")
    a[4, 7] = float("inf")
    a[5, 9] = -float("inf")
    w = torch.ones(512)
    y = rms_norm(a.to(dev), w.to(dev), EPS).cpu()
    _, want = steps(a, None, w)
    np.testing.assert_array_equal(y.numpy(), want)
    q = rms_norm(a.to(dev), w.to(dev), EPS, act_for=GgmlDType.Q4K)
    rows = [0, 1, 2, 6]
    np.testing.assert_array_equal(q.blocks.cpu().numpy()[rows], oracle.quantize_act(12, want[rows]))
    z = rms_norm(torch.zeros(1, 64, device=dev), torch.ones(64, device=dev), 0.0)
    assert z.isnan().all()  # 0 / 0


def test_no_rows(dev):
    from lloom_b200 import GgmlDType, rms_norm

    w = torch.ones(256, device=dev)
    assert rms_norm(torch.empty(0, 256, device=dev), w).shape == (0, 256)
    assert rms_norm(torch.empty(0, 256, device=dev), w, act_for=GgmlDType.Q4K).shape == (0, 256)


def test_stream_and_graph(dev):
    """On a stream of the caller's, and captured: a replay reads what the inputs hold then."""
    from lloom_b200 import GgmlDType, rms_norm

    a, r, w = (t.to(dev) for t in inputs(8, 4, 1024, torch.float16))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y, h = rms_norm(a, w, EPS, r)
    s.synchronize()
    want = rms_norm(a, w, EPS, r)
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, h = rms_norm(a, w, EPS, r, act_for=GgmlDType.Q4K)
        v = q.dequantize()
    b = inputs(9, 4, 1024, torch.float16)[0].to(dev)
    a.copy_(b)
    g.replay()
    torch.cuda.synchronize()
    want_q, want_h = rms_norm(b, w, EPS, r, act_for=GgmlDType.Q4K)
    assert torch.equal(q.blocks, want_q.blocks) and torch.equal(h, want_h) and torch.equal(v, want_q.dequantize())


@pytest.mark.parametrize("fmt", ["Q4_0", "Q5_0", "Q8_0", "Q4K", "Q5K", "Q6K"])
@pytest.mark.parametrize("m,n,k", [(1, 192, 1024), (1, 64, 12544), (2, 192, 1024), (5, 200, 2048), (8, 96, 16384), (9, 128, 1024), (130, 256, 512), (200, 136, 1024)])
def test_products_of_blocks(dev, fmt, m, n, k):
    """A product of blocks has the bits of the product of the values they were made from."""
    from lloom_b200 import GgmlDType, QActs, QMatMul, QTensor
    from lloom_b200.quantized import quantize_weights_host

    dt = getattr(GgmlDType, fmt)
    rng = np.random.default_rng(m + n)
    w = QTensor.from_data(quantize_weights_host(rng.standard_normal((n, k)).astype(np.float32) * np.float32(0.02), dt), dt, (n, k), dev)
    mm = QMatMul.from_qtensor(w)
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(dev)
    acts = QActs.quantize(x, dt)
    assert torch.equal(mm.forward_quantized(acts), mm.forward(x))
    for t in (torch.float16, torch.bfloat16):
        y = mm.forward_quantized(acts, t)
        assert y.dtype == t and torch.equal(y, mm.forward(x).to(t))
    three = QActs(acts.blocks.view(1, m, -1), acts.dtype)
    assert mm.forward_quantized(three).shape == (1, m, n)
    if m > 8 and w.storage.build_prefill_image(w.shape):
        assert torch.equal(mm.forward_quantized(acts), mm.forward(x))


@pytest.mark.parametrize("fmt", ["Q8_0", "Q4K", "Q6K", "Q5_0"])
@pytest.mark.parametrize("m", [1, 2, 3, 8])
def test_decode_step(dev, fmt, m):
    """A layer's way through the operators: norm to blocks, grouped q|k|v, residual, norm, SwiGLU on the stores, down -- the
    bits of the same step on values."""
    from lloom_b200 import GgmlDType, QMatMul, QTensor, rms_norm
    from lloom_b200.quantized import forward_group, quantize_weights_host

    dt, h, kv, f = getattr(GgmlDType, fmt), 1024, 256, 2048
    rng = np.random.default_rng(m)

    def mat(n, k):
        w = quantize_weights_host(rng.standard_normal((n, k)).astype(np.float32) * np.float32(0.02), dt)
        return QMatMul.from_qtensor(QTensor.from_data(w, dt, (n, k), dev))

    q, k, v, gate, up, down = mat(h, h), mat(kv, h), mat(kv, h), mat(f, h), mat(f, h), mat(h, f)
    x = torch.from_numpy(rng.standard_normal((m, h)).astype(np.float32)).to(dev)
    r = torch.from_numpy(rng.standard_normal((m, h)).astype(np.float32)).to(dev)
    w = torch.from_numpy((1 + 0.1 * rng.standard_normal(h)).astype(np.float32)).to(dev)
    y, s = rms_norm(x, w, EPS, r)
    acts, s2 = rms_norm(x, w, EPS, r, act_for=dt)
    assert torch.equal(s, s2)
    want, got = forward_group([q, k, v], y), forward_group([q, k, v], acts)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert torch.equal(got[0], q.forward_quantized(acts)) and torch.equal(got[1], k.forward_quantized(acts))
    y2, s = rms_norm(got[0], w, EPS, s)
    acts2, _ = rms_norm(got[0], w, EPS, s2, act_for=dt)
    hidden = up.forward_mul_into(y2, gate.forward_silu(y2))
    g2 = forward_group([gate], acts2, stores=[1])[0]
    forward_group([up], acts2, stores=[2], outs=[g2])
    assert torch.equal(hidden, g2)
    assert torch.equal(down.forward(hidden), down.forward(g2))


@pytest.mark.parametrize("k", [64, 1000, 4099, 40000])
def test_stream_updated_in_place(dev, k):
    """The C entry with h in the residual's own buffer, rows of x further apart, and weights of another type."""
    from lloom_b200 import _lib

    L = _lib.lib()
    a, r, w = inputs(k, 5, k, torch.float16, torch.float32)
    x = torch.zeros(5, k + 24, dtype=torch.float16, device=dev)
    x[:, :k] = a.to(dev)
    h, y = r.to(dev), torch.empty(5, k, dtype=torch.float16, device=dev)
    wd = w.to(dev)
    assert L.lloom_b200_rms_norm(x.data_ptr(), h.data_ptr(), wd.data_ptr(), 1, 0, EPS, 5, k, k + 24, k, h.data_ptr(), y.data_ptr(), 1,
                                 torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(h.cpu(), steps(a, r, w)[0])
    check_values(y, a, r, w)


@pytest.mark.parametrize("x", ["f16", "f32"])
@pytest.mark.parametrize("m,k", [(700, 1000), (600, 4097), (640, 8192), (600, 8200), (1500, 40), (9, 72)])
def test_many_rows(dev, m, k, x):
    """Two pieces per thread, rows that share a CTA, rows off the boundary among many."""
    from lloom_b200 import rms_norm

    a, r, w = inputs(m + k, m, k, TYPES[x])
    y, h = rms_norm(a.to(dev), w.to(dev), EPS, r.to(dev))
    assert torch.equal(h.cpu(), steps(a, r, w)[0])
    check_values(y, a, r, w)
    # from a base off the boundary, alike for all
    z = torch.zeros(2, m * k + 3, dtype=a.dtype, device=dev)
    z[0, 3:], z[1, 3:] = a.view(-1).to(dev), r.view(-1).to(dev)
    y2, h2 = rms_norm(z[0, 3:].view(m, k), w.to(dev), EPS, z[1, 3:].view(m, k))
    assert torch.equal(y, y2) and torch.equal(h, h2)


@pytest.mark.parametrize("m,k,act", [(70001, 32, "Q8_0"), (70001, 256, "Q4K"), (140003, 9, None), (70001, 520, None)])
def test_rows_past_a_grid(dev, m, k, act):
    """More than 65535 rows, rows that share a CTA among them; as in two halves."""
    import lloom_b200 as lb

    a, r, w = (t.to(dev) for t in inputs(m + k, m, k, torch.bfloat16))
    kind = None if act is None else getattr(lb.GgmlDType, act)
    y, h = lb.rms_norm(a, w, EPS, r, act_for=kind)
    cut = m // 2
    parts = [lb.rms_norm(a[s], w, EPS, r[s], act_for=kind) for s in (slice(0, cut), slice(cut, m))]
    assert torch.equal(h, torch.cat([p[1] for p in parts])) and torch.equal(h, (a.float() + r.float()).bfloat16())
    if act is None:
        assert torch.equal(y, torch.cat([p[0] for p in parts]))
    else:
        assert torch.equal(y.blocks, torch.cat([p[0].blocks for p in parts]))
        assert torch.equal(y.dequantize(), torch.cat([p[0].dequantize() for p in parts]))


@pytest.mark.parametrize("act", [None, "Q4K"])
def test_offsets_past_32_bits(dev, act):
    """A stream of more than 2^31 elements: its last rows as its first ones."""
    import lloom_b200 as lb

    a, r, w = (t.to(dev) for t in inputs(5, 64, 16384, torch.bfloat16))
    reps = 2 ** 31 // (64 * 16384) + 1
    kind = None if act is None else getattr(lb.GgmlDType, act)
    y, h = lb.rms_norm(a.repeat(reps, 1), w, EPS, r.repeat(reps, 1), act_for=kind)
    y1, h1 = lb.rms_norm(a, w, EPS, r, act_for=kind)
    if act is not None:
        y, y1 = y.blocks, y1.blocks
    for got, want in ((y, y1), (h, h1)):
        assert torch.equal(got[:64], want) and torch.equal(got[-64:], want)
        assert (got.view(reps, 64, -1)[::97] == want).all()


@pytest.mark.parametrize("m", [1, 2, 3])
def test_group_into_destinations(dev, m):
    """Destinations of a group: matrices, columns of a wider one, more dimensions, a vector for one row; over values and over blocks."""
    from lloom_b200 import GgmlDType, QMatMul, QTensor, rms_norm
    from lloom_b200.quantized import forward_group, quantize_weights_host

    rng = np.random.default_rng(m)
    mats = []
    for n in (96, 33):
        w = quantize_weights_host(rng.standard_normal((n, 512)).astype(np.float32), GgmlDType.Q4K)
        mats.append(QMatMul.from_qtensor(QTensor.from_data(w, GgmlDType.Q4K, (n, 512), dev)))
    x, w = torch.randn(m, 512, device=dev), torch.ones(512, device=dev)
    for y in (rms_norm(x, w), rms_norm(x, w, act_for=GgmlDType.Q4K)):
        want = forward_group(mats, y)
        wide = torch.full((m, 200), 7.0, device=dev)
        kinds = [[torch.empty(m, 96, device=dev), torch.empty(m, 33, device=dev)], [wide[:, 3:99], wide[:, 120:153]],
                 [torch.empty(1, m, 96, device=dev), torch.empty(m, 1, 33, device=dev)]]
        if m == 1:
            kinds.append([torch.empty(96, device=dev), torch.empty(33, device=dev)])
        for outs in kinds:
            got = forward_group(mats, y, outs=outs)
            for a, b, o in zip(want, got, outs):
                assert b is o and torch.equal(a, b.reshape(a.shape))
        assert (wide[:, :3] == 7).all() and (wide[:, 99:120] == 7).all() and (wide[:, 153:] == 7).all()


def test_group_into_destinations_of_odd_strides(dev):
    """An extent of 1 may have any stride: it does not say how far rows are apart."""
    from lloom_b200 import GgmlDType, QMatMul, QTensor
    from lloom_b200.quantized import forward_group, quantize_weights_host

    w = quantize_weights_host(np.random.default_rng(0).standard_normal((64, 512)).astype(np.float32), GgmlDType.Q4K)
    mm = QMatMul.from_qtensor(QTensor.from_data(w, GgmlDType.Q4K, (64, 512), dev))
    x, buf = torch.randn(3, 512, device=dev), torch.zeros(1000, device=dev)
    want = forward_group([mm], x)[0]
    out = buf.as_strided((3, 1, 64), (64, 200, 1))
    assert out.is_contiguous()
    assert torch.equal(forward_group([mm], x, outs=[out])[0].view(3, 64), want) and not buf[192:].any()
    one = buf.as_strided((1, 64), (1, 1), 400)
    assert torch.equal(forward_group([mm], x[:1], outs=[one])[0], forward_group([mm], x[:1])[0]) and not buf[464:].any()

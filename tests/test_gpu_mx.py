"""Microscaled 4-bit values: quantisation against the definition (bit for bit), blocks in and out, and the product."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


@pytest.fixture(scope="module")
def dev(cuda_lib):
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def quantize(v):
    """Codes [.., k/32, 32] and scale bytes [.., k/32] of f64 values, from the definition (numpy)."""
    v = np.asarray(v, np.float64).reshape(*v.shape[:-1], -1, 32)
    bad = ~np.isfinite(v).all(-1)
    amax = np.abs(np.where(np.isfinite(v), v, 0)).max(-1)
    _, e = np.frexp(amax)
    e = np.where(amax > 0, np.clip(e - 1 - 2, -127, 127), -127)
    with np.errstate(invalid="ignore"):
        r = np.ldexp(np.abs(v), -e[..., None])
        dist = np.abs(r[..., None] - GRID)
        dist = np.where(np.isnan(dist), np.inf, dist)
    best = dist.min(-1, keepdims=True)
    tie = dist == best
    odd = np.arange(8) % 2
    code = np.where(tie, np.arange(8) + 100 * odd, 1000).argmin(-1)  # the even code of a tie
    code = np.where(r >= 6, 7, code)
    code = np.where(np.signbit(v), code + 8, code)
    code = np.where(bad[..., None], 0, code)
    return code.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def pack(codes, scales):
    """17-byte blocks."""
    return np.concatenate([scales[..., None], codes[..., :16] | (codes[..., 16:] << 4)], -1).reshape(*codes.shape[:-2], -1).astype(np.uint8)


def values(codes, scales):
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v * s[..., None]).reshape(*codes.shape[:-2], -1)


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("x", TYPES)
@pytest.mark.parametrize("n,k", [(1, 32), (3, 64), (7, 96), (130, 256), (5, 288), (129, 2080), (2, 4096)])
def test_quantize(dev, n, k, x):
    from lloom_b200 import MxTensor

    v = (normal(n * k, n, k) * torch.exp2(torch.randint(-12, 12, (n, 1), generator=torch.Generator().manual_seed(1)).float())).to(TYPES[x])
    t = MxTensor.quantize(v.to(dev))
    codes, scales = quantize(v.double().numpy())
    assert t.shape == (n, k) and t.data() == pack(codes, scales).tobytes()
    want = values(codes, scales)
    np.testing.assert_array_equal(t.dequantize().cpu().numpy(), want)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(t.dequantize_f16().cpu().numpy(), want.astype(np.float16))


def test_quantize_borders(dev):
    """Every border between two codes and its neighbours, saturation, zeros of both signs, subnormals, the range's ends, NaN and infinity."""
    from lloom_b200 import MxTensor

    edge = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9999995], np.float32)
    row = np.concatenate([edge, np.nextafter(edge, np.float32(0)), np.nextafter(edge, np.float32(9)).clip(max=7.9999995), [4.0, -0.0]]).astype(np.float32)
    rows = [row, -row, row * np.float32(2.0 ** -100), row * np.float32(2.0 ** 124), np.zeros(32, np.float32),
            np.full(32, 1e-45, np.float32), np.linspace(-1e-38, 1e-38, 32, dtype=np.float32), np.full(32, 3.4028235e38, np.float32)]
    for bad in (np.nan, np.inf, -np.inf):
        r = row.copy()
        r[7] = bad
        rows.append(r)
    v = np.stack(rows)
    codes, scales = quantize(v)
    t = MxTensor.quantize(torch.from_numpy(v).to(dev))
    got = np.frombuffer(t.data(), np.uint8).reshape(len(rows), 17)
    want = pack(codes, scales)
    np.testing.assert_array_equal(got[:, 0], want[:, 0])
    np.testing.assert_array_equal(got, want)
    np.testing.assert_array_equal(t.dequantize().cpu().numpy(), values(codes, scales).astype(np.float32))


def test_blocks_in_and_out(dev):
    """Any bytes are blocks: every scale and code survives the way through the image; bytes, arrays, CPU and GPU tensors."""
    from lloom_b200 import MxTensor

    rng = np.random.default_rng(3)
    for n, k in ((1, 32), (200, 288), (128, 256)):
        raw = rng.integers(0, 256, (n, k // 32 * 17), dtype=np.uint8)
        for data in (raw.tobytes(), raw, torch.from_numpy(raw), torch.from_numpy(raw).to(dev)):
            t = MxTensor.from_data(data, (n, k), dev)
            assert t.data() == raw.tobytes()
        blk = raw.reshape(n, k // 32, 17)
        want = values(np.concatenate([blk[..., 1:] & 15, blk[..., 1:] >> 4], -1), blk[..., 0])
        np.testing.assert_array_equal(t.dequantize().cpu().numpy(), want.astype(np.float32))


def whole(seed, rows, k):
    """Values that quantize to themselves with the scale 1: multiples of 1/2 up to 6 with a 4 or more in every block."""
    rng = np.random.default_rng(seed)
    v = rng.choice(GRID, (rows, k)) * rng.choice([-1.0, 1.0], (rows, k))
    v[:, ::32] = rng.choice([-6.0, -4.0, 4.0, 6.0], (rows, k // 32))
    return torch.from_numpy(v.astype(np.float32))


@pytest.mark.parametrize("m", [1, 2, 8, 16, 17, 33, 64, 100, 128, 129, 200, 256, 257, 300, 600])
@pytest.mark.parametrize("n,k", [(1, 32), (130, 256), (100, 320), (385, 2080)])
def test_product_exact(dev, m, n, k):
    """Sums of multiples of 1/4 below 2^22 are exact in f32: the product has no tolerance."""
    from lloom_b200 import MxMatMul, MxTensor

    w, x = whole(n, n, k), whole(m + 1000, m, k)
    mm = MxMatMul.from_tensor(MxTensor.quantize(w.to(dev)))
    want = x.double() @ w.double().T
    y = mm.forward(x.to(dev))
    assert y.dtype == torch.float32 and torch.equal(y.cpu().double(), want)
    for t in (torch.float16, torch.bfloat16):
        y = mm.forward(x.to(t).to(dev))  # up to 6 in steps of 1/2: exact in either
        assert y.dtype == t and torch.equal(y.cpu(), want.to(t))


def check_product(y, x, w_values):
    """|y - exact| <= (steps) * 2^-23 * sum |a w| + the rounding of y's type: an f32 sum of k / 64 partial results per part of K, each
    addition off by at most one unit in the last place of a value below the sum of magnitudes (the tensor core may truncate)."""
    a = torch.from_numpy(values(*quantize(x.double().cpu().numpy()))).to(y.device)
    w = w_values.double()
    want, mag = a @ w.T, a.abs() @ w.abs().T
    tol = (x.shape[-1] / 64 + 8) * 2.0 ** -23 * mag
    if y.dtype != torch.float32:
        tol = tol + (want.abs() + tol) * torch.finfo(y.dtype).eps / 2 + torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("x", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1024, 4096), (8, 3000, 4096), (5, 257, 14336), (37, 4096, 2080), (77, 5000, 2080), (150, 640, 5120), (512, 1024, 2048), (700, 300, 1024)])
def test_product(dev, m, n, k, x):
    from lloom_b200 import MxMatMul, MxTensor

    w = MxTensor.quantize((normal(n, n, k) * 0.02 * torch.exp2(torch.randint(-3, 4, (n, k), generator=torch.Generator().manual_seed(2)).float())).to(dev))
    a = (normal(m + 7, m, k) * torch.exp2(torch.randint(-4, 4, (m, k), generator=torch.Generator().manual_seed(3)).float())).to(TYPES[x]).to(dev)
    mm = MxMatMul.from_tensor(w)
    y = mm.forward(a)
    assert y.shape == (m, n) and y.dtype == a.dtype
    check_product(y, a, w.dequantize())
    assert torch.equal(y, mm.forward(a))  # the parts of K meet in a fixed order
    assert torch.equal(mm.forward(a.view(1, m, k)).view(m, n), y)


def test_bad_values_stay_in_their_rows(dev):
    """A NaN or an infinity makes its own output row NaN, one in the weights its output column; others are untouched."""
    from lloom_b200 import MxMatMul, MxTensor

    w, x = whole(1, 200, 512), whole(2, 40, 512)
    want = x.double() @ w.double().T
    x[3, 100], x[17, 0] = float("nan"), float("-inf")
    w[150, 511] = float("inf")
    y = MxMatMul.from_tensor(MxTensor.quantize(w.to(dev))).forward(x.to(dev)).cpu().double()
    rows = torch.zeros(40, 200, dtype=torch.bool)
    rows[[3, 17]] = True
    rows[:, 150] = True
    assert y[rows].isnan().all() and torch.equal(y[~rows], want[~rows])
    # rows of zeros: scale 2^-127, sums zero
    z = MxMatMul.from_tensor(MxTensor.quantize(torch.zeros(3, 64, device=dev))).forward(torch.zeros(2, 64, device=dev))
    assert torch.equal(z, torch.zeros(2, 3, device=dev))


def test_unaligned_input_and_streams(dev):
    from lloom_b200 import MxMatMul, MxTensor

    w, x = whole(4, 64, 256).to(dev), whole(5, 3, 256).to(dev)
    mm = MxMatMul.from_tensor(MxTensor.quantize(w))
    want = mm.forward(x)
    off = torch.zeros(3 * 256 + 1, device=dev)
    off[1:] = x.view(-1)
    assert torch.equal(mm.forward(off[1:].view(3, 256)), want)
    assert MxTensor.quantize(off[1:].view(3, 256)).data() == MxTensor.quantize(x).data()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for i in range(32):
        with torch.cuda.stream(streams[i % 4]):
            got.append(mm.forward(x))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_chain_and_graph(dev):
    """Products in a chain (each reads the one before, overlapped launches on and off), captured and replayed with other inputs."""
    import lloom_b200 as lb
    from lloom_b200 import _lib

    L = _lib.lib()
    mats = [lb.MxMatMul.from_tensor(lb.MxTensor.quantize((normal(i, 512, 512) * 0.06).to(dev))) for i in range(6)]

    def chain(v):
        for mm in mats:
            v = mm.forward(v)
        return v

    x = normal(50, 4, 512).to(dev)
    before = L.lloom_b200_set_launch_overlap(0)
    try:
        want = chain(x)
        for mode in (1, -1):
            L.lloom_b200_set_launch_overlap(mode)
            for _ in range(5):
                assert torch.equal(chain(x), want)
    finally:
        L.lloom_b200_set_launch_overlap(before)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = chain(x)
    other = normal(51, 4, 512).to(dev)
    x.copy_(other)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, chain(other))
    assert lb.quantized.device_status() == 0


def test_beside_other_products(dev):
    """Between products that take all of tensor memory, on one stream."""
    from lloom_b200 import GgmlDType, MxMatMul, MxTensor, QMatMul, QTensor
    from lloom_b200.quantized import device_status, quantize_weights_host

    rng = np.random.default_rng(0)
    q = QMatMul.from_qtensor(QTensor.from_data(quantize_weights_host(rng.standard_normal((512, 512)).astype(np.float32) * np.float32(0.02), 12), 12, (512, 512), dev))
    assert q.qtensor.dtype() == GgmlDType.Q4K
    mm = MxMatMul.from_tensor(MxTensor.quantize((normal(1, 512, 512) * 0.06).to(dev)))
    x = normal(2, 200, 512).to(dev)
    a = q.forward(x)
    b = mm.forward(a)
    c = q.forward(b)
    torch.cuda.synchronize()
    for _ in range(20):
        assert torch.equal(q.forward(mm.forward(q.forward(x))), c)
    torch.cuda.synchronize()
    assert device_status() == 0 and math.isfinite(float(c.abs().max()))


def test_gguf_tensor(dev):
    """MXFP4 blocks of a file, to a product."""
    import io

    from lloom_b200 import MxMatMul, MxTensor
    from lloom_b200 import gguf_file as G

    w, x = whole(6, 40, 96), whole(7, 3, 96)
    f = io.BytesIO()
    G.write(f, [], [("w", G.MXFP4, (40, 96), pack(*quantize(w.double().numpy())).tobytes())])
    f.seek(0)
    t = G.Content.read(f).tensor(f, "w", dev)
    assert isinstance(t, MxTensor) and t.shape == (40, 96)
    assert torch.equal(MxMatMul.from_tensor(t).forward(x.to(dev)).cpu().double(), x.double() @ w.double().T)


def test_graphs_side_by_side(dev):
    """Two graphs captured on one stream, replayed together on others: neither touches the other's activations."""
    from lloom_b200 import MxMatMul, MxTensor

    mats = [MxMatMul.from_tensor(MxTensor.quantize(whole(i, 4096, 4096).to(dev))) for i in (1, 2)]
    xs = [whole(i + 5, 100, 4096).to(dev) for i in (1, 2)]
    want = [mm.forward(x) for mm, x in zip(mats, xs)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for mm, x in zip(mats, xs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append([mm.forward(x) for _ in range(4)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(30):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, y) for y in o)


@pytest.mark.parametrize("m", [3, 40, 200])
@pytest.mark.parametrize("y_type", [0, 1, 30])
def test_c_entry_row_distance_and_types(dev, m, y_type):
    """Rows of outputs further apart than they are long, results of another type than the activations; what lies between stays."""
    from lloom_b200 import _lib

    L = _lib.lib()
    n, k, ldy = 130, 512, 137
    w, x = whole(1, n, k).to(dev), whole(2, m, k).half().to(dev)
    image = torch.zeros(L.lloom_b200_mx_image_bytes(n, k), dtype=torch.uint8, device=dev)
    ws = torch.empty(L.lloom_b200_mx_workspace_bytes(m, n, k), dtype=torch.uint8, device=dev)
    t = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}[y_type]
    y = torch.full((m, ldy), 77.0, dtype=t, device=dev)
    stream = torch.cuda.current_stream().cuda_stream
    assert L.lloom_b200_mx_quantize(w.data_ptr(), 0, n, k, image.data_ptr(), image.numel(), stream) == 0
    assert L.lloom_b200_mx_fwd(image.data_ptr(), x.data_ptr(), 1, y.data_ptr(), y_type, m, n, k, ldy, ws.data_ptr(), ws.numel(), stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(y[:, :n].cpu(), (x.cpu().double() @ w.cpu().double().T).to(t))
    assert (y[:, n:] == 77).all()


def test_plans_agree(dev):
    """The kernels for few rows, for some and for pairs of CTAs, and their ways of cutting K and the rows: one row's bits where sums are exact."""
    from lloom_b200 import MxMatMul, MxTensor

    for n, k in ((300, 8192), (1100, 16384)):
        w, x = whole(n, n, k), whole(3, 520, k)
        mm = MxMatMul.from_tensor(MxTensor.quantize(w.to(dev)))
        want = (x.double() @ w.double().T).float()
        for m in (1, 2, 4, 16, 17, 65, 128, 129, 250, 384, 520):
            assert torch.equal(mm.forward(x[:m].to(dev)).cpu(), want[:m]), (n, k, m)


@pytest.mark.parametrize("m,n,k", [(70001, 3, 32), (33000, 130, 96), (1, 70001, 32), (300, 40001, 64)])
def test_many_rows(dev, m, n, k):
    """More rows than a grid's second dimension has, on either side."""
    from lloom_b200 import MxMatMul, MxTensor

    w, x = whole(1, n, k), whole(2, m, k)
    t = MxTensor.quantize(w.to(dev))
    assert torch.equal(t.dequantize().cpu(), w)
    got = MxMatMul.from_tensor(t).forward(x.to(dev))
    assert torch.equal(got.double(), x.to(dev).double() @ w.to(dev).double().T)
    assert torch.equal(MxTensor.quantize(x.to(dev)).dequantize().cpu(), x)
    again = MxTensor.from_data(t.data(), (n, k), dev)
    assert torch.equal(again.dequantize().cpu(), w)


@pytest.mark.parametrize("m,n,k", [(33000, 66000, 32), (40, 1100000, 4096)])
def test_offsets_past_32_bits(dev, m, n, k):
    """More than 2^31 outputs; an image of more than 2^31 bytes: rows that repeat, at the end as at the beginning."""
    from lloom_b200 import MxMatMul, MxTensor

    w, x = whole(1, 100, k), whole(2, 40, k)
    mm = MxMatMul.from_tensor(MxTensor.quantize(w.to(dev).bfloat16().repeat(n // 100, 1)))
    y = mm.forward(x.to(dev).bfloat16().repeat(m // 40, 1))
    want = (x.double() @ w.double().T).bfloat16().to(dev)
    for rows in (slice(0, 40), slice(m - 40, m)):
        for cols in (slice(0, 100), slice(n - 100, n)):
            assert torch.equal(y[rows, cols], want)
    assert (y.view(m // 40, -1)[:: max(1, m // 400)] == y[:40].reshape(-1)).all()


@pytest.mark.parametrize("m", [1, 40])
def test_tensor_dropped_while_another_stream_reads_it(dev, m):
    """Its memory goes to others only when that stream has finished with it."""
    import lloom_b200 as lb

    w, x = torch.randn(1024, 4096, device=dev), torch.randn(m, 4096, device=dev)
    t = lb.MxTensor.quantize(w)
    size = t._native.to_blocks().shape[0] // 128 * 16 * (128 * 128 + 1024)
    want = [lb.MxMatMul(t).forward(x), t.dequantize(), t._native.to_blocks()]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for use, ref in zip((lambda t: lb.MxMatMul(t).forward(x), lambda t: t.dequantize(), lambda t: t._native.to_blocks()), want):
        with torch.cuda.stream(side):
            torch.cuda._sleep(40_000_000)
            got = use(t)
        del t
        others = [torch.full((size,), 0x77, dtype=torch.uint8, device=dev) for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(got, ref)
        del others
        t = lb.MxTensor.quantize(w)
        torch.cuda.synchronize()

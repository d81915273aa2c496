"""The draw of the next token against the definition in 64 bits and more: the same token, and its probability."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LAST = float(np.nextafter(np.float32(1), np.float32(0)))


@pytest.fixture(scope="module")
def dev(cuda_lib):
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def draw(l, u, t, k, p, mp):
    """One row, from the definition: (token, probability)."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    top = l.max()
    if top == -np.inf:
        return -1, 0.0
    if not t > 0:
        return int(l.argmax()), 1.0
    order = np.argsort(-l, kind="stable")
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(l == top, 1.0, np.exp((l - top) / t))
    w = np.where(np.isnan(w), 0, w).astype(np.longdouble)
    n = len(l) if k <= 0 else min(k, len(l))
    sums = np.cumsum(w[order[:n]])
    length = n
    if p < 1:
        length = min(n, 1 + int(np.searchsorted(sums, np.longdouble(p) * sums[-1], side="left")))
    if mp > 0:
        length = min(length, max(1, int((w[order[:n]] >= mp).sum())))
    at = np.sort(order[:length])
    sums = np.cumsum(w[at])
    j = min(int(np.searchsorted(sums, np.longdouble(u) * sums[-1], side="right")), length - 1)
    while w[at[j]] == 0:  # u at the end: the last with a weight
        j -= 1
    return int(at[j]), float(w[at[j]] / sums[-1])


def check(dev, logits, u, t=1.0, k=0, p=1.0, mp=0.0):
    """Tokens equal the definition's; probabilities within the rounding to f32 and of the fixed-point sum (2^-44 per token)."""
    import lloom_b200 as lb

    rows = logits.shape[0]
    args = [torch.tensor(v, dtype=torch.int32 if i == 1 else torch.float32, device=dev) if isinstance(v, (list, np.ndarray)) else v
            for i, v in enumerate((t, k, p, mp))]
    u = np.asarray(u, np.float32)
    ids, probs = lb.sample(logits.to(dev), torch.from_numpy(u).to(dev), *args)
    assert ids.dtype == torch.int64 and probs.dtype == torch.float32 and ids.shape == (rows,)
    ids, probs, host = ids.cpu().numpy(), probs.cpu().numpy(), logits.float().numpy()
    per = [np.broadcast_to(np.asarray(v, np.float32 if isinstance(v, (list, np.ndarray)) else np.float64), (rows,)) for v in (t, k, p, mp)]
    for i in range(rows):
        want, prob = draw(host[i], np.float64(u[i]), np.float64(per[0][i]), int(per[1][i]), np.float64(per[2][i]), np.float64(per[3][i]))
        assert ids[i] == want, (i, ids[i], want, prob)
        assert abs(probs[i] - prob) <= prob * (2.0 ** -24 + host.shape[1] * 2.0 ** -44 + 1e-12), (i, probs[i], prob)


def rand(seed, b, v, dtype=torch.float32, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(b, v, generator=g) * scale
    x.scatter_add_(1, torch.randint(0, v, (b, min(v, 24)), generator=g), 4 + 3 * torch.randn(b, min(v, 24), generator=g).abs())
    return x.to(dtype), torch.rand(b, generator=g).numpy()


SETTINGS = [dict(), dict(t=0.7), dict(k=1), dict(k=40, p=0.95, mp=0.05, t=0.8), dict(p=0.9), dict(p=0.999, t=1.5), dict(mp=0.02), dict(k=300, p=0.5),
            dict(k=2000, t=2.0), dict(k=2000, p=0.99, t=2.0), dict(p=0.0), dict(t=0.0), dict(t=50.0), dict(t=50.0, p=0.7), dict(t=50.0, k=777, p=0.9), dict(t=1e-3, k=5)]


@pytest.mark.parametrize("x", TYPES)
@pytest.mark.parametrize("v", [1, 2, 31, 1000, 4096, 4097, 32769, 50257])
def test_settings(dev, v, x):
    for i, s in enumerate(SETTINGS):
        logits, u = rand(v + i, 5, v, TYPES[x])
        check(dev, logits, u, **s)


@pytest.mark.parametrize("x", TYPES)
@pytest.mark.parametrize("v", [128256, 327680])
def test_large(dev, v, x):
    for i, s in enumerate(SETTINGS):
        logits, u = rand(v + i, 2, v, TYPES[x])
        check(dev, logits, u, **s)


@pytest.mark.parametrize("v", [64, 5000, 40000])
def test_equal_logits(dev, v):
    """All equal, and two values only: more ties than are ranked; the filters cut by index."""
    u = np.linspace(0, LAST, 7).astype(np.float32)
    flat = torch.full((7, v), -1.25)
    two = torch.where(torch.rand(7, v, generator=torch.Generator().manual_seed(1)) < 0.5, 1.0, 0.25)
    for logits in (flat, two):
        for s in (dict(), dict(k=v // 3), dict(p=0.37), dict(k=v // 2 + 1, p=0.8), dict(t=0.0), dict(mp=1.0), dict(k=3), dict(p=0.9, t=0.01)):
            check(dev, logits, u, **s)


def test_close_logits(dev):
    """Values one unit in the last place apart around zero and far from it: one bucket holds them all, their bits tell them apart."""
    v = 9000
    g = torch.Generator().manual_seed(2)
    near = torch.randn(3, v, generator=g) * 1e-4
    far = 100 + torch.randint(0, 600, (3, v), generator=g) * 2.0 ** -17
    for logits in (near, far):
        for s in (dict(k=500), dict(p=0.31), dict(k=5000, p=0.5), dict(k=8999)):
            check(dev, logits, np.array([0.1, 0.5, 0.93]), **s)


def test_masks_and_specials(dev):
    """-infinity, the type's lowest value, NaN, +infinity, rows with one token and with none."""
    v = 5000
    logits, u = rand(3, 12, v)
    logits[0, 10:] = -float("inf")
    logits[1, ::2] = torch.finfo(torch.float32).min
    logits[2] = -float("inf")
    logits[3] = -float("inf")
    logits[3, 4999] = -7.0
    logits[4, 100] = float("nan")
    logits[5] = float("nan")
    logits[6, [7, 70, 700]] = float("inf")
    logits[7] = torch.finfo(torch.float32).min
    logits[8, 1:] = torch.finfo(torch.float32).min
    logits[9] = torch.finfo(torch.float32).max
    logits[10, 3] = torch.finfo(torch.float32).max
    for s in (dict(), dict(t=0.0), dict(k=3), dict(k=4000, p=0.9), dict(p=0.5), dict(mp=0.1), dict(k=20, p=0.8, mp=0.01, t=0.3)):
        check(dev, logits, u, **s)
    low = logits.half()
    low[1, ::2] = torch.finfo(torch.float16).min
    check(dev, low, u, k=100, p=0.9)


def test_uniform_numbers_at_the_ends(dev):
    logits, _ = rand(4, 4, 3000)
    for s in (dict(), dict(k=17), dict(p=0.6)):
        check(dev, logits, np.array([0.0, LAST, 1e-30, 0.5]), **s)
    import lloom_b200 as lb

    ids, _ = lb.sample(logits.to(dev), torch.tensor([1.0, 5.0, float("nan"), -1.0], device=dev), top_k=9)
    kept = [sorted(np.argsort(-logits[i].numpy(), kind="stable")[:9]) for i in range(4)]
    assert ids.tolist() == [kept[0][-1], kept[1][-1], kept[2][0], kept[3][0]]


def test_settings_per_row(dev):
    b, v = 24, 20000
    logits, u = rand(5, b, v)
    rng = np.random.default_rng(0)
    t = rng.uniform(0.2, 2.0, b).astype(np.float32)
    t[3] = 0
    k = rng.integers(0, 400, b).astype(np.int32)
    k[[1, 2]] = [0, v + 5]
    p = rng.uniform(0.3, 1.0, b).astype(np.float32)
    p[4] = 1.0
    mp = (rng.uniform(0, 0.1, b) * (rng.random(b) < 0.5)).astype(np.float32)
    check(dev, logits, u, t, k, p, mp)
    check(dev, logits, u, t=t, p=0.9)
    # outside the range: the range's end
    check(dev, logits[:4], u[:4], t=np.array([-1.0, 1.0, 1.0, 1.0], np.float32), k=np.array([3, -7, 0, 2], np.int32),
          p=np.array([0.5, 2.0, -1.0, 0.5], np.float32), mp=np.array([0, 0, -3.0, 0], np.float32))


def test_frequencies(dev):
    """Evenly spaced uniform numbers draw every token as often as its probability says, to within one draw."""
    import lloom_b200 as lb

    v, n = 50, 4096
    row = torch.randn(v, generator=torch.Generator().manual_seed(6))
    u = (torch.arange(n) + 0.5) / n
    ids, _ = lb.sample(row.expand(n, v).contiguous().to(dev), u.to(dev), temperature=0.9)
    got = torch.bincount(ids.cpu(), minlength=v).double()
    want = torch.softmax(row.double() / 0.9, 0) * n
    assert ((got - want).abs() <= 1).all()


def test_rows_apart_shapes_and_streams(dev):
    import lloom_b200 as lb

    logits, u = rand(7, 6, 3001, torch.bfloat16)
    wide = torch.zeros(6, 5000, dtype=torch.bfloat16, device=dev)
    wide[:, 7:3008] = logits.to(dev)
    ud = torch.from_numpy(u).to(dev)
    want = lb.sample(logits.to(dev), ud, 0.9, 50, 0.9)
    got = lb.sample(wide[:, 7:3008], ud, 0.9, 50, 0.9)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    three = lb.sample(logits.to(dev).view(2, 3, 3001), ud.view(2, 3), 0.9, 50, 0.9)
    assert three[0].shape == (2, 3) and torch.equal(three[0].view(-1), want[0])
    one = lb.sample(logits[0].to(dev), ud[0], 0.9, 50, 0.9)
    assert one[0].shape == () and one[0] == want[0][0]
    none = lb.sample(torch.empty(0, 10, device=dev), torch.empty(0, device=dev))
    assert none[0].shape == (0,)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = lb.sample(logits.to(dev), ud, 0.9, 50, 0.9)
    s.synchronize()
    assert torch.equal(got[0], want[0])


def test_output_head_then_draw_captured(dev):
    """The output head's product and the draw behind it in one graph, replayed with other hidden states and numbers."""
    import lloom_b200 as lb
    from lloom_b200.quantized import quantize_weights_host

    v, h, b = 8000, 512, 3
    rng = np.random.default_rng(1)
    w = quantize_weights_host(rng.standard_normal((v, h)).astype(np.float32) * np.float32(0.1), 14)
    head = lb.QMatMul.from_qtensor(lb.QTensor.from_data(w, lb.GgmlDType.Q6K, (v, h), dev))
    norm = torch.ones(h, device=dev)
    x, u = torch.randn(b, h, device=dev), torch.rand(b, device=dev)

    def step():
        logits = head.forward_quantized(lb.rms_norm(x, norm, act_for=lb.GgmlDType.Q6K))
        return lb.sample(logits, u, 0.8, 100, 0.9), logits

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        (ids, probs), logits = step()
    for i in range(3):
        x.copy_(torch.randn(b, h, device=dev))
        u.copy_(torch.rand(b, device=dev))
        g.replay()
        torch.cuda.synchronize()
        got = (ids.clone(), probs.clone())
        (want, want_p), _ = step()
        assert torch.equal(got[0], want) and torch.equal(got[1], want_p)
        for r in range(b):
            assert got[0][r] == draw(logits[r].cpu().numpy(), float(u[r]), 0.8, 100, 0.9, 0.0)[0]


def test_c_entry(dev):
    """Rows apart, no probabilities wanted, settings of every kind; streams side by side."""
    from lloom_b200 import _lib

    L = _lib.lib()
    b, v = 6, 5003
    logits, u = rand(9, b, v, torch.float16)
    wide = torch.full((b, v + 13), 60000.0, dtype=torch.float16, device=dev)
    wide[:, :v] = logits.to(dev)
    ud, k = torch.from_numpy(u).to(dev), torch.full((b,), 33, dtype=torch.int32, device=dev)
    want = [draw(logits[i].float().numpy(), np.float64(u[i]), 0.9, 33, 0.8, 0.0)[0] for i in range(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = [torch.full((b + 1,), -5, dtype=torch.int64, device=dev) for _ in range(32)]
    torch.cuda.synchronize()
    for i, ids in enumerate(outs):
        assert L.lloom_b200_sample(wide.data_ptr(), 1, b, v, v + 13, ud.data_ptr(), None, 0.9, k.data_ptr(), 0, None, 0.8, None, 0.0, ids.data_ptr(),
                                   None, streams[i % 4].cuda_stream) == 0
    torch.cuda.synchronize()
    for ids in outs:
        assert ids.tolist() == want + [-5]


def test_least_temperature(dev):
    """Temperatures down to 2^-120 are computed with, below that the first of the largest is taken; a temperature without end draws evenly."""
    logits = torch.tensor([[1.0, 3.0, 3.0, 2.0]] * 3)
    u = np.array([0.1, 0.6, 0.9])
    check(dev, logits, u, t=2.0 ** -119)
    check(dev, logits, u, t=float("inf"))
    import lloom_b200 as lb

    ids, probs = lb.sample(logits.to(dev), torch.from_numpy(u.astype(np.float32)).to(dev), temperature=2.0 ** -121)
    assert ids.tolist() == [1, 1, 1] and probs.tolist() == [1.0, 1.0, 1.0]


@pytest.mark.parametrize("n", [1, 2, 33, 64, 65, 200, 257, 511, 512, 513, 700])
def test_tokens_of_one_bucket(dev, n):
    """The border among n tokens that lie within 1/64 of one another, behind 300 others: sorted, or searched by ranges; for weights and for counts."""
    rng = np.random.default_rng(n)
    v = 300 + n + 20000
    rows = []
    for ties in (False, True):
        near = 2.0 + rng.random(n) * 0.006
        if ties:
            near = 2.0 + rng.integers(0, 3, n) * 0.002
        row = np.concatenate([4 + rng.random(300), near, -6 - rng.random(20000)])
        rows.append(row[rng.permutation(v)])
    logits = torch.from_numpy(np.array(rows).astype(np.float32))
    w = np.exp(np.sort(logits.double().numpy(), 1)[:, ::-1] - logits.double().max(1).values.numpy()[:, None])
    u = np.array([0.999, 0.97])
    for share in (0.1, 0.5, 0.93):
        at = 300 + int(share * n)
        check(dev, logits, u, k=at + 1)
        check(dev, logits, u, p=(w[:, :at].sum(1) + 0.5 * w[:, at]) / w.sum(1))
        check(dev, logits, u, k=at + 1, p=0.9999, mp=1e-6)


@pytest.mark.parametrize("b,v", [(70001, 5), (3000, 517), (300, 9000)])
def test_more_rows_than_fit_at_once(dev, b, v):
    """Settings of their own for every row; rows that repeat give the same token."""
    import lloom_b200 as lb

    base, u = rand(b, 50, v)
    reps = -(-b // 50)
    logits, u = base.repeat(reps, 1)[:b], np.tile(u, reps)[:b]
    t = np.tile(np.linspace(0.0, 2.0, 50, dtype=np.float32), reps)[:b]
    k = np.tile(np.arange(50, dtype=np.int32), reps)[:b]
    p = np.tile(np.linspace(0.3, 1.0, 50, dtype=np.float32), reps)[:b]
    check(dev, logits[:50], u[:50], t=t[:50], k=k[:50], p=p[:50])
    args = [torch.from_numpy(a).to(dev) for a in (u, t, k, p)]
    ids, probs = lb.sample(logits.to(dev), *args)
    for out in (ids, probs):
        full = torch.cat([out, out[-50:]])
        assert torch.equal(out[50:], out[:-50]) and full.shape[0] == b + 50


def test_logits_past_32_bits(dev):
    """A batch of more than 2^31 logits: its last rows as its first ones."""
    import lloom_b200 as lb

    base, u = rand(1, 8, 50257, torch.float16)
    reps = 2 ** 31 // (8 * 50257) + 2
    logits = base.to(dev).repeat(reps, 1)
    assert logits.numel() > 2 ** 31
    ids, probs = lb.sample(logits, torch.from_numpy(u).to(dev).repeat(reps), top_p=0.8)
    assert (ids.view(reps, 8) == ids[:8]).all() and (probs.view(reps, 8) == probs[:8]).all()
    check(dev, base, u, p=0.8)


FAR_SETTINGS = [dict(), dict(k=1), dict(k=40), dict(p=0.9), dict(mp=0.05), dict(k=40, p=0.9, mp=0.05)]


def check_drawn(dev, logits, u, t, s):
    """As check, and every row with a finite logit gives a token and a probability."""
    import lloom_b200 as lb

    check(dev, logits, u, t=t, **s)
    ids, probs = lb.sample(logits.to(dev), torch.from_numpy(np.asarray(u, np.float32)).to(dev), t, s.get("k", 0), s.get("p", 1.0), s.get("mp", 0.0))
    assert (ids >= 0).all() and (probs > 0).all() and (probs <= 1).all()


@pytest.mark.parametrize("v", [300, 20000])
@pytest.mark.parametrize("t", [1e-6, 1e-9, 1e-12, 1e-14, 1e-15, 1e-16, 1e-17, 1e-18, 1e-20, 1e-22, 1e-24, 1e-26])
def test_small_temperatures(dev, t, v):
    """Largest logits with full mantissas over temperatures from 10^-6 to 10^-26: the largest's own weight is 1, and ties of it share the draw."""
    for x in TYPES.values():
        logits, u = rand(v, 4, v, x)
        logits[1, [7, 70, 270]] = logits[1].max()
        logits[2] = -logits[2].abs() - 3.3
        logits[3, v // 2:] = logits[3].max()
        for s in FAR_SETTINGS:
            check_drawn(dev, logits, u, t, s)


@pytest.mark.parametrize("x", ["f32", "bf16"])
@pytest.mark.parametrize("e", range(50, 92, 3))
def test_logits_far_from_zero(dev, e, x):
    """Largest logits around 2^50 to 2^90 at ordinary temperatures, of either sign, alone, tied, and rows of one finite mask value."""
    v = 3000
    base, u = rand(e, 5, v)
    logits = base * 2.0 ** (e - 3)
    logits[1, [7, 70, 700]] = logits[1].max()
    logits[2] = -logits[2].abs() - 1.234567 * 2.0 ** e
    logits[3] = -1.234567 * 2.0 ** e
    logits[4] = 1.234567 * 2.0 ** e
    for t in (0.7, 0.8, 1.0):
        for s in FAR_SETTINGS:
            check_drawn(dev, logits.to(TYPES[x]), u, t, s)


@pytest.mark.parametrize("value", [-1e16, -1e18, -1e20, 1e18, 1e20])
def test_rows_of_one_far_value(dev, value):
    logits, u = torch.full((3, 4000), value), np.array([0.0, 0.4, LAST])
    for t in (0.7, 1.0):
        for s in FAR_SETTINGS:
            check_drawn(dev, logits, u, t, s)
            check_drawn(dev, logits.bfloat16(), u, t, s)


@pytest.mark.parametrize("top,t", [(20.0, 3e-7), (100.0, 1e-6), (1000.0, 1e-5), (3e7, 0.9), (1e12, 3e4), (1e-30, 1e-31)])
def test_close_logits_far_from_zero(dev, top, t):
    """Logits within some temperatures of the largest, which is 10^7 temperatures and more from zero: weights as exact as near zero."""
    v = 6000
    g = torch.Generator().manual_seed(9)
    ulp = float(np.spacing(np.float32(top)))
    steps = torch.randint(0, max(2, int(25 * t / ulp)), (4, v), generator=g).double()
    logits = (top - steps * ulp).float()
    u = np.array([0.05, 0.31, 0.62, 0.97])
    for s in (dict(), dict(k=100), dict(k=3000), dict(p=0.9), dict(p=0.5, mp=0.01)):
        check_drawn(dev, logits, u, t, s)
        check_drawn(dev, -logits, u, t, s)

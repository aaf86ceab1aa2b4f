"""Sampling against a plain 64-bit form: tokens equal, probabilities to f32
rounding (2^-24) and the 2^-43 units that weights are counted in (half of one,
2^-44 of the largest weight, over a probability's own: below 2^-22 relative for
any token above 2^-22 of it, and 2^-43 absolute)."""
import numpy as np
import pytest

from pagedref import sample

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(torch):
    from grande_b200 import ops
    return ops


TYPES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16"}


def check(torch, ops, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """x [rows, vocab] on the device; settings numbers or host arrays."""
    rows = x.shape[0]
    par = {"temperature": (temperature, torch.float32), "top_k": (top_k, torch.int32),
           "top_p": (top_p, torch.float32), "min_p": (min_p, torch.float32)}
    dev = {k: v if np.isscalar(v) else torch.tensor(v, dtype=t, device=x.device)
           for k, (v, t) in par.items()}
    tok, prob = ops.sample(x, torch.tensor(u, dtype=torch.float32, device=x.device), **dev)
    tok, prob = tok.cpu().numpy(), prob.cpu().numpy()
    h = x.float().cpu().numpy()
    f = {k: np.broadcast_to(np.asarray(v, np.int32 if k == "top_k" else np.float32), rows)
         for k, (v, _) in par.items()}
    for r in range(rows):
        t, p = sample(h[r], np.float32(u[r]), *(f[k][r] for k in par))
        assert tok[r] == t, (r, tok[r], t, prob[r], p, {k: f[k][r] for k in par})
        assert abs(prob[r] - p) <= p * 2.0 ** -22 + 2.0 ** -43, (r, prob[r], p)
    return tok


def logits(torch, rows, vocab, seed, device, dtype="f32", spread=2.5, hot=8):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device=f"cuda:{device}") * spread
    if hot:
        at = torch.randint(0, vocab, (rows, hot), generator=g, device=x.device)
        x.scatter_add_(1, at, torch.rand((rows, hot), generator=g, device=x.device) * 10)
    return x.to(getattr(torch, TYPES[dtype]))


def uniforms(rows, seed):
    u = np.random.default_rng(seed).random(rows).astype(np.float32)
    return np.minimum(u, np.float32(1 - 2.0 ** -24))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [1, 2, 7, 300, 4097, 25000, 56001])
@pytest.mark.parametrize("kw", [
    dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=64, top_p=0.95), dict(top_k=5),
    dict(top_p=0.9), dict(min_p=0.05), dict(top_k=2000, top_p=0.5, min_p=0.01),
    dict(top_k=3000, top_p=0.7, temperature=1.7), dict(top_p=0.999, temperature=0.3),
    dict(top_p=1e-6), dict(min_p=1.0), dict(temperature=50.0, top_p=0.5),
])
def test_settings(device, torch, ops, dtype, vocab, kw):
    x = logits(torch, 6, vocab, vocab, device, dtype)
    check(torch, ops, x, uniforms(6, vocab), **kw)


@pytest.mark.parametrize("dtype,vocab", [("f32", 327680), ("f32", 524288), ("bf16", 524288), ("f16", 262144)])
def test_largest_vocabularies(device, torch, ops, dtype, vocab):
    # 4 rows: clusters of CTAs; 90: one CTA per row, which reads it three times.
    for rows in (4, 90):
        x = logits(torch, rows, vocab, 1, device, dtype)
        for kw in (dict(), dict(top_p=0.9), dict(top_k=100000, top_p=0.95), dict(top_k=50)):
            check(torch, ops, x[:90:23] if rows == 90 else x, uniforms(4, 2), **kw)
        if rows == 90:
            u = torch.tensor(uniforms(90, 2), device=x.device)
            whole = ops.sample(x, u, top_p=0.9)
            for r in range(0, 90, 29):
                one = ops.sample(x[r:r + 1], u[r:r + 1], top_p=0.9)
                assert one[0] == whole[0][r] and one[1] == whole[1][r]


@pytest.mark.parametrize("rows,vocab,dtype", [
    (1, 30000, "f32"), (3, 150001, "bf16"), (20, 60000, "f16"), (80, 45003, "f32"), (2, 70000, "f32")])
@pytest.mark.parametrize("shape", ["flat", "even", "wide", "peak", "two", "steps", "holes"])
def test_top_p_of_whole_rows(device, torch, ops, rows, vocab, dtype, shape):
    """Where the mass is reached: among a few of thousands of logits of a kind,
    beside one or two that hold most of it, among equal ones, between rows of
    -infinity and NaN; alone and with min-p."""
    x = logits(torch, rows, vocab, 5, device, "f32",
               {"flat": 0.004, "even": 0.8, "peak": 0.8, "two": 1.5}.get(shape, 6.0), 0)
    if shape == "peak":
        x[:, 77] = np.log(vocab) + 1.0
    elif shape == "two":
        x[:, ::vocab - 1] = np.log(vocab) + 1.5
    elif shape == "steps":
        x = (x * 3).round() / 3
    elif shape == "holes":
        x[:, ::2] = -np.inf
        x[:, 1::6] = np.nan
    x = x.to(getattr(torch, TYPES[dtype]))
    p = np.resize(np.array([0.9, 0.5, 0.05, 0.999, 0.99999, 0.7], np.float32), rows)
    check(torch, ops, x, uniforms(rows, 3), top_p=p)
    check(torch, ops, x, uniforms(rows, 4), top_p=p, min_p=0.02, temperature=0.7)


@pytest.mark.parametrize("rows", [1, 3, 40, 75, 200])
def test_settings_of_each_row(device, torch, ops, rows):
    rng = np.random.default_rng(rows)
    x = logits(torch, rows, 9000, rows, device)
    pick = lambda *v: rng.choice(v, rows)  # noqa: E731
    check(torch, ops, x, uniforms(rows, rows), pick(0.0, 0.5, 1.0, 2.0).astype(np.float32),
          pick(0, -3, 1, 40, 2500, 9000, 100000).astype(np.int32),
          pick(0.0, 0.3, 0.9, 1.0, 7.0).astype(np.float32),
          pick(-1.0, 0.0, 0.1, 1.0).astype(np.float32))


@pytest.mark.parametrize("values", [1, 2, 3, 40])
@pytest.mark.parametrize("kw", [
    dict(), dict(top_k=64), dict(top_k=2047, top_p=0.5), dict(top_p=0.5), dict(top_p=0.25),
    dict(top_k=6000, top_p=0.75), dict(min_p=0.2), dict(top_k=20000)])
def test_ties(device, torch, ops, values, kw):
    """A row of few distinct values: thresholds fall among equal logits, which
    stay by index, and borders fall on exact multiples."""
    g = torch.Generator(device="cuda").manual_seed(values)
    x = torch.randint(0, values, (8, 30000), generator=g, device=f"cuda:{device}").float() / 8
    u = np.array([0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.1, 0.3, 0.9], np.float32)
    check(torch, ops, x, u, **kw)


def test_masked_infinite_and_nan_logits(device, torch, ops):
    x = logits(torch, 9, 5000, 3, device)
    inf = float("inf")
    x[0] = -inf
    x[1] = float("nan")
    x[2, 1:] = -inf
    x[3, ::2] = float("nan")
    x[4, [7, 900, 4999]] = inf
    x[5, :4990] = -inf
    x[6] = -inf
    x[6, 4999] = -3e38
    x[7] = x[7] * 1e37
    x[8, 5:] = torch.finfo(torch.float32).min
    for kw in (dict(), dict(top_k=3, top_p=0.9), dict(top_p=0.6), dict(top_k=3000), dict(min_p=0.5),
               dict(temperature=1e-40), dict(temperature=1e30)):
        tok = check(torch, ops, x, uniforms(9, 5), **kw)
        assert tok[0] == tok[1] == -1 and tok[2] == 0 and tok[6] == 4999


def test_the_draw_follows_the_uniform_numbers(device, torch, ops):
    """All uniform numbers of a grid: each token as often as its share."""
    x = torch.log(torch.tensor([1.0, 2.0, 4.0, 1.0], device=f"cuda:{device}")).repeat(64, 1)
    u = (np.arange(64) + 0.5) / 64
    tok = check(torch, ops, x, u)
    assert np.bincount(tok).tolist() == [8, 16, 32, 8]


def test_strides_alignment_and_outputs(device, torch, ops):
    wide = logits(torch, 5, 1003, 7, device)
    for lo in range(4):
        check(torch, ops, wide[:, lo:lo + 997], uniforms(5, lo), top_p=0.8)
    half = wide.half()
    for lo in range(8):
        check(torch, ops, half[:, lo:lo + 990], uniforms(5, lo), top_k=30)
    tokens = torch.full((5,), -9, dtype=torch.int32, device=wide.device)
    probs = torch.zeros(5, device=wide.device)
    u = torch.full((5,), 0.5, device=wide.device)
    got = ops.sample(wide, u, tokens=tokens, probs=probs)
    assert got[0] is tokens and got[1] is probs and (tokens >= 0).all() and (probs > 0).all()


def test_repeats_streams_and_graphs(device, torch, ops):
    x = logits(torch, 30, 25000, 8, device, "f16")
    u = torch.rand(30, device=x.device)
    kw = dict(temperature=1.3, top_k=4000, top_p=0.97)
    first = [t.clone() for t in ops.sample(x, u, **kw)]
    for _ in range(5):
        again = ops.sample(x, u, **kw)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    side = torch.cuda.Stream(x.device)
    side.wait_stream(torch.cuda.current_stream(x.device))
    with torch.cuda.stream(side):
        other = ops.sample(x, u, **kw)
    torch.cuda.current_stream(x.device).wait_stream(side)
    assert torch.equal(first[0], other[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, prob = ops.sample(x, u, **kw)
    u.copy_(torch.rand(30, device=x.device))
    graph.replay()
    want = ops.sample(x, u, **kw)
    assert torch.equal(tok, want[0]) and torch.equal(prob, want[1])

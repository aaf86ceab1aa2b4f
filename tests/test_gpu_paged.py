"""The paged append and the paged attention against plain 64-bit forms.

Tolerances count roundings. u is half a step of the 16-bit type (2^-11 f16,
2^-8 bf16). An append output is rounded once: u relative, plus the f32 work
before it (norm, rotation: under 16 roundings of values no larger than the
pair's, 2^-20 of its magnitude). An attention output is rounded once and its
probabilities once: u |out| + u sum p|v|, plus 2^-14 sum p|v| for scores,
exponentials and sums in f32 (a score of magnitude 32 carries 2^-18, the sums
over a few thousand keys less), plus what f16 loses below 2^-14: 2^-25 of the
largest |v| per key, and of the output itself."""
import numpy as np
import pytest

from pagedref import Batch, append, attention

pytestmark = pytest.mark.gpu

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(torch):
    from grande_b200 import ops
    return ops


def dtype_of(torch, name):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def host(t):
    return t.float().cpu().numpy()


def make_cache(torch, dev, b, kvh, hd, dtype, g, fill=float("nan")):
    """Random K/V in the rows that hold tokens, `fill` everywhere else."""
    cache = torch.full((b.n_pages * b.page, 2, kvh, hd), fill, device=dev)
    used = torch.from_numpy(b.used_rows()).to(dev)
    cache[used] = torch.randn((len(used), 2, kvh, hd), generator=g, device=dev)
    return cache.view(b.n_pages, b.page, 2, kvh, hd).to(dtype)


def check_attention(got, q, cache, b, scale, window, dtype):
    exp, mag = attention(host(q)[:b.tokens], host(cache), b, scale, window)
    u = U[dtype]
    keys = max(b.lens + [0]) + max(b.prefix_lens + [0])
    tol = u * np.abs(exp) + (u + 2.0 ** -14) * mag + (keys + 1) * 2.0 ** -25 * 8
    err = np.abs(host(got)[:b.tokens] - exp)
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[bad][:5])


GROUPS = {
    "token": [(37, [(4, 1), (0, 1), (63, 1), (64, 1)])],
    "groups": [(130, [(3, 1), (70, 1)]), (0, [(9, 1)]), (64, [(1, 1)] * 5)],
    "branches": [(70, [(0, 24), (0, 5), (0, 1)]), (3, [(10, 40)])],
    "prompt": [(0, [(0, 150), (20, 33)])],
    "empty": [(20, []), (0, [(5, 0), (5, 1), (0, 0), (2, 3)]), (9, [(0, 0)])],
    "long": [(1500, [(700, 1), (2, 1), (0, 3)]), (500, [(64, 2)])],
}


@pytest.mark.parametrize("hd,heads,kvh", [(256, 8, 2), (256, 4, 1), (512, 8, 2), (128, 6, 2),
                                          (64, 16, 1), (64, 3, 3)])
@pytest.mark.parametrize("name", list(GROUPS))
@pytest.mark.parametrize("dtype,page,window", [("f16", 16, 0), ("bf16", 32, 7), ("f16", 64, 100),
                                               ("f16", 128, 1)])
def test_attention(device, torch, ops, hd, heads, kvh, name, dtype, page, window):
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(hd + heads + page)
    b = Batch(GROUPS[name], page, np.random.default_rng(page + window))
    cache = make_cache(torch, dev, b, kvh, hd, dtype_of(torch, dtype), g)
    q = torch.randn((b.tokens, heads, hd), generator=g, device=dev).to(cache.dtype)
    scale = 1.5 / np.sqrt(hd)
    got = ops.paged_attention(q, cache, b.device(ops, torch, dev), scale=scale, window=window)
    check_attention(got, q, cache, b, np.float32(scale), window, dtype)


@pytest.mark.parametrize("hd,heads,kvh", [(64, 8, 1), (128, 32, 4), (256, 6, 2), (512, 8, 2)])
@pytest.mark.parametrize("groups", [
    [(0, [(0, 900)])],                                         # a prompt: row tiles of 1 key tile on
    [(5 * i, [(i % 4, 1 + i % 3)]) for i in range(400)],       # hundreds of short row tiles
    [(700, [(0, 300), (3, 1), (90, 77)]), (0, [(1, 1)] * 30)]  # cut by several CTAs each
], ids=["prompt", "many", "cut"])
def test_lines_of_many_row_tiles(device, torch, ops, hd, heads, kvh, groups):
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(hd)
    b = Batch(groups, 32, np.random.default_rng(hd))
    cache = make_cache(torch, dev, b, kvh, hd, torch.bfloat16, g)
    q = torch.randn((b.tokens, heads, hd), generator=g, device=dev).to(cache.dtype)
    scale = 1.5 / np.sqrt(hd)
    got = ops.paged_attention(q, cache, b.device(ops, torch, dev), scale=scale)
    check_attention(got, q, cache, b, np.float32(scale), 0, "bf16")


def test_attention_without_groups_equals_one_group_without_prefix(device, torch, ops):
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(5)
    seqs = [(0, [(n, 1) for n in (3, 90, 0, 200, 64)])]
    b = Batch(seqs, 16, np.random.default_rng(1))
    cache = make_cache(torch, dev, b, 2, 256, torch.float16, g)
    q = torch.randn((b.tokens, 8, 256), generator=g, device=dev).half()
    one = ops.paged_attention(q, cache, b.device(ops, torch, dev), scale=0.1)
    b.grouped = False
    none = ops.paged_attention(q, cache, b.device(ops, torch, dev), scale=0.1)
    assert torch.equal(one, none)
    check_attention(none, q, cache, b, np.float32(0.1), 0, "f16")


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("window", [0, 6])
def test_what_a_row_does_not_see_does_not_reach_it(device, torch, ops, hd, window):
    """Infinities and NaN in keys and values of other sequences, of later
    tokens, of rows behind the window and of unused rows."""
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(hd)
    b = Batch([(40, [(5, 1), (70, 6), (2, 1)]), (0, [(30, 1)])], 16, np.random.default_rng(2))
    cache = make_cache(torch, dev, b, 2, hd, torch.float16, g)
    flat = cache.view(-1, 2, 2, hd)
    # The second sequence's third new token, and its whole first 20 tokens'
    # predecessors when a window hides them from its last rows.
    own = b.rows(b.pages[1], b.lens[1])
    flat[own[72], 1, :, 3] = float("inf")
    flat[own[72], 0, 0, 0] = float("nan")
    flat[own[73], 1, 1] = float("nan")
    # A prefix key that only rows of sequence 2 can still see under the window.
    if window:
        flat[b.rows(b.prefix_pages[0], 40)[38], 1, :, 5] = -float("inf")
    q = torch.randn((b.tokens, 4, hd), generator=g, device=dev).half()
    got = host(ops.paged_attention(q, cache, b.device(ops, torch, dev), scale=0.1, window=window))
    with np.errstate(invalid="ignore", over="ignore"):
        exp, _ = attention(host(q), host(cache), b, np.float32(0.1), window)
    finite = np.isfinite(exp)
    assert (np.isfinite(got) == finite).all(), np.argwhere(np.isfinite(got) != finite)[:5]
    assert finite[0].all() and finite[1:3].all() and not finite[4:].all()
    assert np.abs(got - exp)[finite].max() < 5e-3


def test_rows_that_see_nothing_are_zero_and_padding_is_left(device, torch, ops):
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(3)
    b = Batch([(0, [(4, 1), (0, 1), (2, 2)])], 16, np.random.default_rng(3))
    cache = make_cache(torch, dev, b, 1, 256, torch.float16, g)
    q = torch.randn((b.tokens + 3, 2, 256), generator=g, device=dev).half()
    out = torch.full_like(q, 7.0)
    lens = list(b.lens)
    lens[1] = 0  # a query row without a token behind it
    dev_b = b.device(ops, torch, dev, lens=lens)
    ops.paged_attention(q, cache, dev_b, scale=0.1, out=out)
    assert (out[b.tokens:] == 7).all()
    assert (out[1] == 0).all()
    b.lens[1] = 1
    rows = [0, 2, 3]
    exp, _ = attention(host(q)[:b.tokens], host(cache), b, np.float32(0.1), 0)
    assert np.abs(host(out)[rows] - exp[rows]).max() < 5e-3


def test_tables_the_pool_does_not_hold(device, torch, ops):
    """Page ids outside the pool read as zeros, lengths are cut at the tables:
    nothing outside them is touched."""
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(4)
    b = Batch([(20, [(40, 1), (3, 1)])], 16, np.random.default_rng(4))
    cache = make_cache(torch, dev, b, 2, 256, torch.float16, g)
    q = torch.randn((b.tokens, 4, 256), generator=g, device=dev).half()
    pages = b.pages.copy()
    pages[0, 1] = b.n_pages + 1000000
    pages[0, 2] = -2147483648
    got = ops.paged_attention(q, cache, b.device(ops, torch, dev, pages=pages,
                                                 lens=[41 + 5000, 4]), scale=0.1)
    assert torch.isfinite(got).all()
    exp, _ = attention(host(q), host(cache), b, np.float32(0.1), 0)
    assert np.abs(host(got)[1] - exp[1]).max() < 5e-3
    before = cache.clone()
    ops.paged_append(torch.randn((b.tokens, 8 * 256), device=dev), cache,
                     b.device(ops, torch, dev, pages=pages), heads=4)
    changed = (cache.view(torch.int16) != before.view(torch.int16)).flatten(2).any(-1).nonzero()
    want = int(b.pages[1, 0]), 3
    assert changed.tolist() == [list(want)]


def test_strides_streams_and_a_replayed_graph(device, torch, ops):
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(6)
    b = Batch([(100, [(30, 1), (60, 1), (0, 1)])], 32, np.random.default_rng(6))
    cache = make_cache(torch, dev, b, 2, 256, torch.float16, g, fill=0.0)
    wide = torch.randn((b.tokens, 11, 256), generator=g, device=dev).half()
    q = wide[:, 2:10]  # rows further apart than they are long
    held = torch.zeros((b.tokens, 9, 256), device=dev, dtype=torch.float16)
    out = held[:, :8]
    dev_b = b.device(ops, torch, dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        ops.paged_attention(q, cache, dev_b, scale=0.1, out=out)
    torch.cuda.current_stream(dev).wait_stream(side)
    check_attention(out, q, cache, b, np.float32(0.1), 0, "f16")
    assert (held[:, 8] == 0).all()
    # A graph follows the tensors it was captured over: lengths grow.
    ws = torch.empty(ops.paged_attention_workspace(cache, dev_b, b.tokens, 8), dtype=torch.uint8,
                     device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention(q, cache, dev_b, scale=0.1, out=out, workspace=ws)
    for _ in range(2):
        b.lens = [n - 7 if n > 20 else n for n in b.lens]
        dev_b.lens.copy_(torch.tensor(b.lens, dtype=torch.int32))
        graph.replay()
        check_attention(out, q, cache, b, np.float32(0.1), 0, "f16")


@pytest.mark.parametrize("src,dtype", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"),
                                       ("bf16", "bf16")])
@pytest.mark.parametrize("hd,heads,kvh,rot", [(256, 8, 2, 256), (512, 4, 1, 128), (128, 3, 3, 128),
                                              (64, 5, 1, 0), (64, 2, 2, 32)])
@pytest.mark.parametrize("norm,v_norm,offset", [(True, False, 1.0), (False, True, 0.0)])
def test_append(device, torch, ops, src, dtype, hd, heads, kvh, rot, norm, v_norm, offset):
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(hd + heads)
    b = Batch([(131000, [(5, 3), (0, 1), (15, 18)]), (0, [(0, 0), (33, 2)])], 16,
              np.random.default_rng(hd))
    cache = torch.randn((b.n_pages, 16, 2, kvh, hd), generator=g, device=dev).to(
        dtype_of(torch, dtype))
    before = cache.clone()
    qkv = (torch.randn((b.tokens + 2, (heads + 2 * kvh) * hd + 16), generator=g, device=dev) *
           3).to(dtype_of(torch, src))[:, :(heads + 2 * kvh) * hd]
    qn = torch.randn(hd, generator=g, device=dev) * 0.2 if norm else None
    kn = torch.randn(hd, generator=g, device=dev) * 0.2 if norm else None
    freq = ops.rope_frequencies(1e6, hd, rot, scale=2.0, device=dev)
    out = torch.full((b.tokens + 2, heads, hd), 7.0, device=dev, dtype=cache.dtype)
    prefix_pages = np.zeros((2, 131000 // 16 + 1), np.int32)
    dev_b = b.device(ops, torch, dev, prefix_pages=prefix_pages)
    ops.paged_append(qkv, cache, dev_b, heads=heads, q_norm=qn, k_norm=kn, norm_offset=offset,
                     eps=1e-5, v_norm=v_norm, inv_freq=freq if rot else None, q_scale=0.25,
                     out=out)
    exp_q, exp_c = append(host(qkv), host(before), b, heads,
                          None if qn is None else host(qn), None if kn is None else host(kn),
                          offset, 1e-5, v_norm, freq.cpu().numpy(), 0.25)
    assert (out[b.tokens:] == 7).all()
    touched = np.zeros(b.n_pages * 16, bool)
    for s, _, _, rows, i0 in b.sequences():
        touched[b.rows(b.pages[s], b.lens[s])[i0:]] = True
    same = (cache.view(torch.int16) == before.view(torch.int16)).flatten(2).all(-1).flatten()
    assert same.cpu().numpy()[~touched].all()

    def check(got, exp):
        half = np.roll(exp, hd // 2, -1)  # the other value of each rotated pair
        tol = U[dtype] * np.abs(exp) + 2.0 ** -20 * (np.abs(exp) + np.abs(half)) + 2.0 ** -25
        err = np.abs(got - exp)
        assert (err <= tol).all(), (np.argwhere(err > tol)[:4], err[err > tol][:4])

    check(host(out)[:b.tokens], exp_q)
    check(host(cache).reshape(-1, 2, kvh, hd)[touched], exp_c.reshape(-1, 2, kvh, hd)[touched])


def test_append_of_queries_alone_leaves_the_cache(device, torch, ops):
    dev = torch.device("cuda", device)
    b = Batch([(7, [(3, 2), (1, 1)])], 16, np.random.default_rng(9))
    cache = torch.randn((b.n_pages, 16, 2, 2, 256), device=dev).half()
    before = cache.clone()
    qkv = torch.randn((b.tokens, 4 * 256), device=dev)
    dev_b = b.device(ops, torch, dev)
    got = ops.paged_append(qkv, cache, dev_b, heads=4)
    assert torch.equal(cache, before)
    assert torch.equal(got, qkv.half().view(b.tokens, 4, 256))


def test_empty_calls_launch_nothing(device, torch, ops):
    dev = torch.device("cuda", device)
    i32 = dict(dtype=torch.int32, device=dev)
    none = ops.PagedBatch(torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros((0, 1), **i32))
    cache = torch.zeros((1, 16, 2, 1, 64), device=dev).half()
    assert ops.paged_append(torch.zeros((0, 192), device=dev), cache, none, heads=1).numel() == 0
    q = torch.full((2, 1, 64), 3.0, device=dev).half()
    out = torch.full_like(q, 7.0)
    ops.paged_attention(q, cache, none, out=out)
    assert (out == 7).all()


def test_rows_past_32_bits_of_the_pool(device, torch, ops):
    """A pool of 6 GB: rows whose byte and element offsets pass 2^32 and 2^31."""
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(8)
    b = Batch([(30, [(50, 1), (3, 2)])], 16, np.random.default_rng(8))
    n_pages = 100000  # x 16 rows x 2,048 values x 2 bytes
    cache = torch.empty((n_pages, 16, 2, 4, 256), dtype=torch.float16, device=dev)
    up = n_pages - b.n_pages
    cache[up:] = make_cache(torch, dev, b, 4, 256, torch.float16, g)
    dev_b = b.device(ops, torch, dev, pages=b.pages + up, prefix_pages=b.prefix_pages + up)
    qkv = torch.randn((b.tokens, 16 * 256), generator=g, device=dev)
    before = cache[up:].clone()
    q = ops.paged_append(qkv, cache, dev_b, heads=8)
    _, exp_c = append(host(qkv), host(before), b, 8, None, None, 0.0, 0.0, False, np.zeros(0), 1.0)
    used = b.used_rows()
    got_c = host(cache[up:]).reshape(-1, 2048)[used]
    assert np.abs(got_c - exp_c.reshape(-1, 2048)[used]).max() < 4e-3
    out = ops.paged_attention(q, cache, dev_b, scale=0.05)
    check_attention(out, q, cache[up:], b, np.float32(0.05), 0, "f16")


def test_two_graphs_and_two_streams_with_workspaces_of_their_own(device, torch, ops):
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(12)
    b = Batch([(700, [(30, 1)] * 7), (90, [(200, 4)] * 3)], 32, np.random.default_rng(12))
    cache = make_cache(torch, dev, b, 2, 128, torch.float16, g, fill=0.0)
    dev_b = b.device(ops, torch, dev)
    qs = [torch.randn((b.tokens, 8, 128), generator=g, device=dev).half() for _ in range(2)]
    want = [ops.paged_attention(q, cache, dev_b, scale=0.1) for q in qs]
    check_attention(want[0], qs[0], cache, b, np.float32(0.1), 0, "f16")
    graphs, outs = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.paged_attention(q, cache, dev_b, scale=0.1))
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize(dev)
    # The work is cut the same way each time, so the bits are the same.
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_a_first_call_under_capture(device, tmp_path):
    """A process whose first call of each operator is captured."""
    import subprocess
    import sys
    from pathlib import Path
    code = f"""
import torch
from grande_b200 import ops
dev = torch.device("cuda", {device})
torch.cuda.set_device(dev)
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
b = ops.PagedBatch(i32([0, 1, 2]), i32([3, 20]), i32([[0, 1], [2, 3]]))
cache = torch.zeros((4, 16, 2, 1, 256), device=dev).half()
qkv = torch.ones((2, 4 * 256), device=dev)
u = torch.full((2,), 0.5, device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    q = ops.paged_append(qkv, cache, b, heads=2)
    out = ops.paged_attention(q, cache, b)
    tok, prob = ops.sample(out.view(2, 512), u)
graph.replay()
torch.cuda.synchronize()
# The last key of each sequence is the row just appended, the others zeros.
assert out[0].min() > 0.9 and tok.min() >= 0
"""
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_an_output_in_place_is_refused(device, torch, ops):
    dev = torch.device("cuda", device)
    b = Batch([(0, [(3, 1)])], 16, np.random.default_rng(1))
    cache = torch.zeros((b.n_pages, 16, 2, 1, 64), device=dev).half()
    q = torch.zeros((1, 1, 64), device=dev).half()
    with pytest.raises(ops.OmgError, match="out is q"):
        ops.paged_attention(q, cache, b.device(ops, torch, dev), out=q)
    with pytest.raises(ops.OmgError, match="workspace of 256 bytes"):
        ops.paged_attention(q, cache, b.device(ops, torch, dev),
                            workspace=torch.empty(256, dtype=torch.uint8, device=dev))
    with pytest.raises(ops.OmgError, match="out must be"):
        ops.paged_attention(q, cache, b.device(ops, torch, dev), out=q[:, :, :32])
    with pytest.raises(ops.OmgError, match="norm must be 64 contiguous"):
        ops.paged_append(torch.zeros((1, 192), device=dev), cache, b.device(ops, torch, dev),
                         heads=1, q_norm=torch.zeros(32, device=dev))

"""Engine.sample_groups: the tokens sampled on the device from a request's
logits rows equal those sampled on the host from the rows that
evaluate_groups returns, for one group and for several whose rows leave the
device in another order; and the paged operators and the sampling run
together as a decoding loop uses them."""
import numpy as np
import pytest

from grande_b200._lib import OmgError
from grande_b200.engine import BranchTokens, Group, Want
from oracle import oracle as O
from pagedref import Batch, append, attention, sample
from refmodels import RefModel, gemma3, gemma4

pytestmark = pytest.mark.gpu


def requests():
    one = [Group([2, 7, 11, 19, 23], [BranchTokens([5, 6, 9], [0, 2]),
                                      BranchTokens([30, 31], [1])])]
    many = [Group([3, 4, 5, 6], [BranchTokens([7, 8], [1]), BranchTokens([9], [0])]),
            Group([2, 7, 11, 19, 23], [BranchTokens([5, 6, 9], [2, 0, 1])]),
            Group([12, 13], [BranchTokens([14, 15, 16], [0, 2]), BranchTokens([3], [])])]
    return one, many


@pytest.mark.parametrize("config", [gemma3, gemma4])
@pytest.mark.parametrize("per_row", [False, True])
def test_sampled_rows_equal_the_rows_sampled_on_the_host(device, config, per_row):
    eng = RefModel(*config(), 37, O.Q8, O.Q8).engine(64, 16, device)
    one, many = requests()
    # Twice `many`: the second time with a prefix of it resident.
    for groups in (one, many, many):
        n = sum(g.rows() for g in groups)
        rng = np.random.default_rng(n)
        u = rng.random(n).astype(np.float32)
        kw = dict(temperature=0.7, top_k=20, top_p=0.9, min_p=0.01)
        if per_row:
            kw = dict(temperature=rng.choice([0.0, 0.5, 2.0], n), top_k=rng.integers(0, 30, n),
                      top_p=rng.choice([0.5, 1.0], n), min_p=rng.choice([0.0, 0.1], n))
        got = eng.sample_groups(groups, u, **kw)
        rows = eng.evaluate_groups(groups, Want.LOGITS)
        r = 0
        for g, (a, b) in enumerate(zip(got, rows)):
            for s, e, br in zip(a.branches, b.branches, groups[g].branches):
                assert s.tokens.shape == s.probs.shape == (len(br.want),)
                for t, p, row in zip(s.tokens, s.probs, e.rows):
                    f = [np.float32(kw[k][r]) if per_row else np.float32(kw[k])
                         for k in ("temperature", "top_k", "top_p", "min_p")]
                    et, ep = sample(row, u[r], f[0], int(f[1]), f[2], f[3])
                    assert t == et and abs(p - ep) <= ep * 2.0 ** -22
                    r += 1
    assert [x.tokens.tolist() for x in eng.sample(one[0].prefix, one[0].branches, [0.1, 0.2, 0.3],
                                                  temperature=0.0)] == [
        [int(row.argmax()) for row in e.rows]
        for e in eng.evaluate(one[0].prefix, one[0].branches, Want.LOGITS)]
    for args, text in [((one, [0.5]), "uniforms: .1. values for 3 rows"),
                       ((one, 0.5), "a sequence of 3 numbers"), (([], []), "empty request")]:
        with pytest.raises(OmgError, match=text):
            eng.sample_groups(*args)
    with pytest.raises(OmgError, match="top_p: .2. values for 3 rows"):
        eng.sample_groups(one, [0.1, 0.2, 0.3], top_p=[0.5, 0.5])
    eng.close()


def test_a_row_wanted_several_times_is_sampled_each_time(device):
    eng = RefModel(*gemma3(), 37, O.Q8, O.Q8).engine(64, 16, device)
    groups = [Group([2, 7, 11], [BranchTokens([5, 6, 9], [2, 0, 2, 2]), BranchTokens([3], [0, 0])])]
    u = np.array([0.05, 0.5, 0.95, 0.4, 0.99, 0.01], np.float32)
    temperature = np.array([99.0, 1.0, 99.0, 0.0, 50.0, 50.0], np.float32)  # nearly even rows
    got = eng.sample_groups(groups, u, temperature=temperature)[0].branches
    rows = [r for b in eng.evaluate_groups(groups, Want.LOGITS)[0].branches for r in b.rows]
    exp = [sample(r, *x, 0, np.float32(1), np.float32(0)) for r, x in zip(rows, zip(u, temperature))]
    assert [t for b in got for t in b.tokens] == [t for t, _ in exp]
    assert exp[0][0] != exp[2][0] and exp[4][0] != exp[5][0]
    eng.close()


def test_a_decoding_loop(device):
    """Two states, three branches: prompts appended and attended, then tokens
    one at a time, the last output through a projection to logits and sampled;
    every step against the plain forms, and the last ones from a graph."""
    torch = pytest.importorskip("torch")
    from grande_b200 import ops
    dev = torch.device("cuda", device)
    g = torch.Generator(device=dev).manual_seed(11)
    heads, kvh, hd, page, vocab = 4, 2, 64, 16, 500
    rng = np.random.default_rng(11)
    # Room for 4 more tokens per branch: pages are handed out at the end's length.
    full = Batch([(40, [(0, 14), (0, 9)]), (17, [(0, 20)])], page, rng)
    cache = torch.randn((full.n_pages, page, 2, kvh, hd), generator=g, device=dev).half()
    freq = ops.rope_frequencies(1e4, hd, device=dev)
    qn = torch.randn(hd, generator=g, device=dev) * 0.1
    head = torch.randn((heads * hd, vocab), generator=g, device=dev) * 0.2
    lens = [10, 5, 16]  # after the prompts
    host = cache.float().cpu().numpy()

    def step(b, dev_b, qkv):
        q = ops.paged_append(qkv, cache, dev_b, heads=heads, q_norm=qn, k_norm=qn,
                             norm_offset=1.0, inv_freq=freq, q_scale=0.2)
        return q, ops.paged_attention(q, cache, dev_b, window=30)

    def check(b, qkv, q, out):
        nonlocal host
        eq, host = append(qkv.cpu().numpy(), host, b, heads, qn.cpu().numpy(), qn.cpu().numpy(),
                          1.0, 1e-6, False, freq.cpu().numpy(), 0.2)
        assert np.abs(q.float().cpu().numpy() - eq).max() < 2e-3
        host = cache.float().cpu().numpy()  # the rounded rows are what is attended
        eo, _ = attention(q.float().cpu().numpy(), host, b, 1.0, 30)
        assert np.abs(out.float().cpu().numpy() - eo).max() < 5e-3

    b = full
    b.q_start, b.lens, b.tokens = [0, 10, 15, 31], list(lens), 31
    dev_b = b.device(ops, torch, dev)
    dev_b.validate(cache, 31)
    qkv = torch.randn((31, (heads + 2 * kvh) * hd), generator=g, device=dev)
    check(b, qkv, *step(b, dev_b, qkv))
    # One token each: the tables stay, the lengths grow in place.
    b.q_start, b.tokens = [0, 1, 2, 3], 3
    dev_b = b.device(ops, torch, dev)
    qkv = torch.empty((3, (heads + 2 * kvh) * hd), device=dev)
    u = torch.empty(3, device=dev)

    def token():
        q, out = step(b, dev_b, qkv)
        logits = out.float().view(3, -1) @ head
        return q, out, logits, ops.sample(logits, u, top_k=50, top_p=0.9)

    graph = None
    for i in range(4):
        b.lens = [n + 1 for n in b.lens]
        dev_b.lens.copy_(torch.tensor(b.lens, dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=dev))
        u.copy_(torch.rand(3, generator=g, device=dev))
        if i < 2:
            res = token()
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    res = token()
            graph.replay()
        q, out, logits, (tok, prob) = res
        check(b, qkv, q, out)
        for r in range(3):
            et, ep = sample(logits[r].cpu().numpy(), u[r].item(), 1.0, 50, np.float32(0.9), 0.0)
            assert tok[r].item() == et and abs(prob[r].item() - ep) <= ep * 2.0 ** -22

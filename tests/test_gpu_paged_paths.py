"""Paths of the paged operators that depend on the size of a batch, and calls at
the edge of what they take, against plain 64-bit forms; tolerances as derived in
test_gpu_paged.py."""
import numpy as np
import pytest

from pagedref import Batch, append, attention
from test_gpu_paged import (U, check_attention, dtype_of, host, make_cache, ops,  # noqa: F401
                            torch)

pytestmark = pytest.mark.gpu


def device_of(torch, device):  # noqa: F811
    return torch.device("cuda", device)


def test_head_counts_refused(device, torch, ops):  # noqa: F811
    dev = device_of(torch, device)
    b = Batch([(0, [(3, 1)])], 16, np.random.default_rng(1))
    cache = torch.zeros((b.n_pages, 16, 2, 2, 64), device=dev).half()
    # As wide as 3 heads: -1 query heads and 2 + 2 of the cache.
    for heads in (-1, 0):
        with pytest.raises(ops.OmgError, match=f"paged_append: heads {heads}"):
            ops.paged_append(torch.zeros((1, (heads + 4) * 64), device=dev), cache,
                             b.device(ops, torch, dev), heads=heads)


# Up to 148 tokens a block takes one, up to 740 two, beyond that four.
@pytest.mark.parametrize("tokens", [147, 149, 301, 740, 803, 2501])
@pytest.mark.parametrize("hd,heads,kvh,src,dtype,rot", [
    (64, 3, 1, "f32", "f16", 64), (512, 2, 1, "bf16", "bf16", 128), (128, 16, 4, "f16", "f16", 128),
    (256, 4, 1, "f32", "bf16", 0)])
def test_appends_of_many_tokens(device, torch, ops, tokens, hd, heads, kvh, src, dtype, rot):  # noqa: F811
    dev = device_of(torch, device)
    rng = np.random.default_rng(tokens + hd)
    g = torch.Generator(device=dev).manual_seed(tokens + hd)
    # Ragged sequences, empty ones among them, 3 rows of padding.
    new = []
    while sum(new) < tokens - 3:
        new += [0] * int(rng.integers(0, 3)) + [min(int(rng.integers(1, 90)), tokens - 3 - sum(new))]
    seqs = [(int(rng.integers(0, 300)), n) for n in new]
    b = Batch([(5000, seqs[::2]), (0, []), (77, seqs[1::2])], 256, rng)
    cache = torch.randn((b.n_pages, 256, 2, kvh, hd), generator=g, device=dev).to(
        dtype_of(torch, dtype))
    before = cache.clone()
    qkv = torch.randn((tokens, (heads + 2 * kvh) * hd), generator=g, device=dev).to(
        dtype_of(torch, src))
    qn, kn = (torch.randn(hd, generator=g, device=dev) * 0.2 for _ in range(2))
    freq = ops.rope_frequencies(1e4, hd, rot, device=dev)
    out = torch.full((tokens, heads, hd), 7.0, device=dev, dtype=cache.dtype)
    ops.paged_append(qkv, cache, b.device(ops, torch, dev), heads=heads, q_norm=qn, k_norm=kn,
                     norm_offset=1.0, v_norm=True, inv_freq=freq if rot else None, q_scale=0.25,
                     out=out)
    exp_q, exp_c = append(host(qkv), host(before), b, heads, host(qn), host(kn), 1.0, 1e-6, True,
                          freq.cpu().numpy(), 0.25)
    assert b.tokens == tokens - 3 and (out[b.tokens:] == 7).all()
    touched = np.zeros(b.n_pages * 256, bool)
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


def run_attention(torch, ops, dev, groups, page, hd, heads, kvh, dtype, window, seed, scale=None):  # noqa: F811
    g = torch.Generator(device=dev).manual_seed(seed)
    b = Batch(groups, page, np.random.default_rng(seed))
    cache = make_cache(torch, dev, b, kvh, hd, dtype_of(torch, dtype), g)
    q = torch.randn((b.tokens, heads, hd), generator=g, device=dev).to(cache.dtype)
    scale = scale or 1.5 / np.sqrt(hd)
    got = ops.paged_attention(q, cache, b.device(ops, torch, dev), scale=scale, window=window)
    check_attention(got, q, cache, b, np.float32(scale), window, dtype)


# A row tile holds 128 query heads of a KV head: these hold 33 to 129 runs.
@pytest.mark.parametrize("hd,heads,kvh", [(64, 2, 2), (128, 3, 1), (256, 2, 1), (512, 1, 1)])
@pytest.mark.parametrize("prefix", [0, 150])
@pytest.mark.parametrize("window", [0, 9, 170])
def test_many_sequences_in_a_row_tile(device, torch, ops, hd, heads, kvh, prefix, window):  # noqa: F811
    dev = device_of(torch, device)
    rng = np.random.default_rng(hd + prefix)
    one = [(int(rng.integers(0, 60)), 1) for _ in range(70)]
    gaps = [x for s in one for x in [s] + [(4, 0)] * int(rng.integers(0, 4))]
    some = [(int(rng.integers(0, 60)), int(rng.integers(0, 4))) for _ in range(160)]
    for i, groups in enumerate([[(prefix, one)], [(prefix, gaps), (20, one[:33])], [(prefix, some)],
                                [(prefix, one * 2)]]):
        run_attention(torch, ops, dev, groups, 16, hd, heads, kvh, "f16", window, hd + i)


@pytest.mark.parametrize("heads,kvh", [(64, 1), (128, 1), (256, 2), (43, 1), (65, 1), (127, 1)])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("groups", [[(70, [(5, 1)])], [(70, [(5, 1), (0, 3), (40, 2)]), (0, [(9, 4)])]],
                         ids=["one", "some"])
def test_many_query_heads_of_a_kv_head(device, torch, ops, heads, kvh, hd, groups):  # noqa: F811
    run_attention(torch, ops, device_of(torch, device), groups, 64, hd, heads, kvh, "bf16", 0, heads + hd)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [0, 100])
def test_pages_of_256_rows(device, torch, ops, hd, window):  # noqa: F811
    run_attention(torch, ops, device_of(torch, device),
                  [(600, [(255, 1), (256, 1), (30, 260), (0, 1)]), (256, [(511, 2)])], 256, hd, 4, 2,
                  "f16", window, hd)


def test_elements_past_32_bits_of_the_pool(device, torch, ops):  # noqa: F811
    """A pool of 9.2 GB: its last rows lie past 2^32 elements."""
    dev = device_of(torch, device)
    g = torch.Generator(device=dev).manual_seed(8)
    b = Batch([(30, [(50, 1), (3, 2)])], 16, np.random.default_rng(8))
    n_pages = 140000  # x 16 rows x 2,048 values
    cache = torch.empty((n_pages, 16, 2, 4, 256), dtype=torch.float16, device=dev)
    up = n_pages - b.n_pages
    assert up * 16 * 2048 > 2 ** 32
    cache[up:] = make_cache(torch, dev, b, 4, 256, torch.float16, g)
    dev_b = b.device(ops, torch, dev, pages=b.pages + up, prefix_pages=b.prefix_pages + up)
    qkv = torch.randn((b.tokens, 16 * 256), generator=g, device=dev)
    before = cache[up:].clone()
    q = ops.paged_append(qkv, cache, dev_b, heads=8)
    _, exp = append(host(qkv), host(before), b, 8, None, None, 0.0, 0.0, False, np.zeros(0), 1.0)
    used = b.used_rows()
    got, exp = (x.reshape(-1, 2048)[used] for x in (host(cache[up:]), exp))
    # Rounded once.
    assert (np.abs(got - exp) <= U["f16"] * np.abs(exp) + 2.0 ** -25).all()
    out = ops.paged_attention(q, cache, dev_b, scale=0.05)
    check_attention(out, q, cache[up:], b, np.float32(0.05), 0, "f16")


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [0, 7])
@pytest.mark.parametrize("what", ["no pages", "no tokens", "some without tokens"])
@pytest.mark.parametrize("seqs", [3, 200])
def test_rows_without_own_keys_see_the_prefix(device, torch, ops, hd, window, what, seqs):  # noqa: F811
    """A row sees its group's prefix up to its own position also where its own
    keys are cut: by a table without pages, or by a length below its query rows
    (own index -1: the prefix's last token is at its position)."""
    dev = device_of(torch, device)
    g = torch.Generator(device=dev).manual_seed(hd)
    b = Batch([(40, [(0, 1)] * seqs), (0, [(0, 1)]), (21, [(0, 1)] * 2)], 16, np.random.default_rng(hd))
    cache = make_cache(torch, dev, b, 2, hd, torch.float16, g)
    q = torch.randn((b.tokens, 4, hd), generator=g, device=dev).half()
    pages, lens = b.pages, np.array(b.lens)
    if what == "no pages":
        pages = b.pages[:, :0]
    else:
        lens[::1 if what == "no tokens" else 3] = 0
    got = host(ops.paged_attention(q, cache, b.device(ops, torch, dev, pages=pages, lens=lens),
                                   scale=0.1, window=window))
    # As queries of the prefix alone, or of prefix and own key.
    flat = host(cache).reshape(-1, 2, 2, hd).astype(np.float64)
    exp, mag = np.zeros(q.shape), np.zeros(q.shape)
    for s, plen, grp, rows, _ in b.sequences():
        pos = plen + lens[s] - 1
        kv = flat[np.concatenate([b.rows(b.prefix_pages[grp], plen),
                                  b.rows(b.pages[s], lens[s] if what != "no pages" else 0)])]
        kv = kv[max(0, pos - window + 1) if window else 0:]
        for h in range(4 if len(kv) else 0):
            z = kv[:, 0, h // 2] @ host(q)[rows[0], h].astype(np.float64) * np.float32(0.1)
            p = np.exp(z - z.max())
            p /= p.sum()
            exp[rows[0], h], mag[rows[0], h] = p @ kv[:, 1, h // 2], p @ np.abs(kv[:, 1, h // 2])
    tol = U["f16"] * np.abs(exp) + (U["f16"] + 2.0 ** -14) * mag + 42 * 2.0 ** -25 * 8
    err = np.abs(got - exp)
    assert (err <= tol).all(), (np.argwhere(err > tol)[:5], err[err > tol][:5])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd,heads", [(64, 128), (128, 128), (256, 64), (512, 64)])
@pytest.mark.parametrize("at", [0, 20000, 39999])
def test_many_small_weights_beside_a_large_one(device, torch, ops, dtype, hd, heads, at):  # noqa: F811
    """40,000 keys of e^-17.5 (2^-25.2) of one key's weight each hold 1e-3 of the
    sum together. Every row tile's keys are in one or two CTAs' ranges. P of the
    type: the large one's V is zero, so u per small one, f16 below 2^-14 half of
    2^-24, of a weight of 2^8 for the largest."""
    dev = device_of(torch, device)
    keys, tokens = 40000, 400
    b = Batch([(keys, [(0, 1)] * tokens)], 256, np.random.default_rng(1))
    cache = torch.zeros((b.n_pages, 256, 2, 1, hd), device=dev).to(dtype_of(torch, dtype))
    cache[:, :, 1] = 1.0
    flat = cache.view(-1, 2, 1, hd)
    large = int(b.rows(b.prefix_pages[0], keys)[at])
    flat[large, 0, 0, 0], flat[large, 1] = 5.0, 0.0
    q = torch.zeros((tokens, heads, hd), device=dev).to(cache.dtype)
    q[..., 0] = 3.5
    got = host(ops.paged_attention(q, cache, b.device(ops, torch, dev), scale=1.0))
    exp = keys * np.exp(-17.5) / (1 + keys * np.exp(-17.5))  # with its own key, without the large one
    u = U[dtype]
    tol = 2 * u * exp + 2.0 ** -14 * exp + (keys * 2.0 ** -33 if dtype == "f16" else 0)
    assert np.abs(got - exp).max() <= tol, (np.abs(got - exp).max(), tol)

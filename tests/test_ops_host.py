"""What the operators on device memory refuse, on the CPU: the C entry points
before they touch a device, PagedBatch's shapes and its validation."""
import ctypes as C

import numpy as np
import pytest

from grande_b200 import _lib as L

torch = pytest.importorskip("torch")
from grande_b200 import ops  # noqa: E402

P = 4096  # an aligned address that is never followed


def cache(**kw):
    f = dict(rows=P, n_pages=8, page_rows=16, kv_heads=2, head_dim=256, dtype=0)
    f.update(kw)
    return L.PagedCacheC(**f)


def batch(**kw):
    f = dict(q_start=P, lens=P, pages=P, group_start=P, prefix_lens=P, prefix_pages=P, n_seqs=3,
             n_groups=1, max_pages=4, max_prefix_pages=4)
    f.update(kw)
    return L.PagedBatchC(**f)


def append_args(**kw):
    f = dict(qkv=P, qkv_stride=12 * 256, qkv_dtype=2, tokens=5, heads=8, has_kv=1, q_out=P,
             q_stride=8 * 256, q_norm=P, k_norm=P, v_norm=0, norm_offset=0.0, eps=1e-6, q_scale=1.0,
             inv_freq=P, n_freq=128)
    f.update(kw)
    return L.AppendArgsC(**f)


def attention_args(**kw):
    f = dict(q=P, q_stride=8 * 256, out=P, out_stride=8 * 256, tokens=5, heads=8, window=0,
             scale=1.0)
    f.update(kw)
    return L.AttentionArgsC(**f)


def refused(rc, text):
    assert rc == -1
    msg = L.lib().omg_last_error().decode()
    assert text in msg, msg


def call_append(c=None, b=None, a=None, device=0):
    return L.lib().omg_paged_append(device, C.byref(c or cache()), C.byref(b or batch()),
                                    C.byref(a or append_args()), None)


@pytest.mark.parametrize("kw,text", [
    (dict(rows=0), "cache rows is null"),
    (dict(rows=P + 8), "cache rows is not 16-byte aligned"),
    (dict(dtype=2), "cache dtype 2"),
    (dict(head_dim=96), "head_dim 96"),
    (dict(kv_heads=0), "kv_heads 0"),
    (dict(page_rows=8), "page of 8 rows"),
    (dict(page_rows=48), "page of 48 rows"),
    (dict(page_rows=512), "page of 512 rows"),
    (dict(n_pages=0), "0 pages"),
    (dict(n_pages=1 << 27), "pages of 16 rows"),
])
def test_caches_refused(kw, text):
    refused(call_append(c=cache(**kw)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(n_seqs=-1), "negative batch size"),
    (dict(q_start=0), "q_start is null"),
    (dict(lens=P + 2), "lens is not 4-byte aligned"),
    (dict(pages=0), "pages is null"),
    (dict(group_start=0), "group_start is null"),
    (dict(max_pages=1 << 27), "rows per sequence"),
])
def test_batches_refused(kw, text):
    refused(call_append(b=batch(**kw)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(heads=0), "heads 0"),
    (dict(tokens=-1), "negative batch size"),
    (dict(qkv_dtype=1), "qkv dtype 1"),
    (dict(qkv=P + 4), "qkv is not 16-byte aligned"),
    (dict(q_out=0), "q_out is null"),
    (dict(qkv_stride=11 * 256), "qkv stride"),
    (dict(qkv_stride=12 * 256 + 1), "qkv stride"),
    (dict(q_stride=7 * 256), "q stride"),
    (dict(n_freq=129), "129 rotated pairs"),
    (dict(inv_freq=0), "inv_freq is null"),
    (dict(k_norm=P + 4), "k_norm is not 16-byte aligned"),
    (dict(eps=-1.0), "eps"),
    (dict(q_scale=float("nan")), "q_scale"),
])
def test_appends_refused(kw, text):
    refused(call_append(a=append_args(**kw)), text)


@pytest.mark.parametrize("kw,text", [
    (dict(scale=0.0), "scale 0"),
    (dict(scale=float("inf")), "scale inf"),
    (dict(window=-1), "window -1"),
    (dict(window=(1 << 30) + 1), "window"),
    (dict(heads=9), "9 query heads over 2 KV heads"),
    (dict(heads=258), "258 query heads over 2 KV heads"),
])
def test_attentions_refused(kw, text):
    rc = L.lib().omg_paged_attention(0, C.byref(cache()), C.byref(batch()),
                                     C.byref(attention_args(**kw)), P, 1 << 30, None)
    refused(rc, text)


# 8 heads over 2 KV heads: 32 tokens to a row tile. The first two fill the plan
# kernel's shared memory; the others' line of key tiles would pass 2^29.
@pytest.mark.parametrize("b,tokens", [
    (dict(n_seqs=30000), 5),
    (dict(n_seqs=1), 1 << 21),
    (dict(n_seqs=32, max_pages=1 << 26), 32),
    (dict(n_seqs=1, max_pages=1 << 20), 1 << 16),
    (dict(n_seqs=1, max_prefix_pages=1 << 20), 1 << 16),
])
def test_batches_past_the_plan_refused(b, tokens):
    b = batch(**b)
    rc = L.lib().omg_paged_attention(0, C.byref(cache()), C.byref(b),
                                     C.byref(attention_args(tokens=tokens)), P, 1 << 40, None)
    refused(rc, "split the batch")
    assert L.lib().omg_paged_attention_workspace(0, C.byref(cache()), C.byref(b), tokens, 8) == 0


def test_null_structs_and_devices_refused():
    lib = L.lib()
    refused(call_append(device=-1), "device -1")
    refused(call_append(device=64), "device 64")
    refused(lib.omg_paged_append(0, None, C.byref(batch()), C.byref(append_args()), None),
            "cache is null")
    refused(lib.omg_paged_append(0, C.byref(cache()), None, C.byref(append_args()), None),
            "batch is null")
    refused(lib.omg_paged_append(0, C.byref(cache()), C.byref(batch()), None, None), "args is null")
    refused(lib.omg_paged_attention(0, C.byref(cache()), C.byref(batch()), None, P, 0, None),
            "args is null")


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def test_batch_shapes():
    good = dict(q_start=i32([0, 1, 3]), lens=i32([4, 5]), pages=i32([[0], [1]]))
    ops.PagedBatch(**good)
    for kw, text in [
        (dict(q_start=i32([0, 1])), r"q_start is \[2\], expected \[3\]"),
        (dict(lens=torch.tensor([4, 5])), "lens must be a contiguous int32"),
        (dict(pages=i32([[0, 1]])), r"pages is \[1, 2\]"),
        (dict(prefix_lens=i32([1])), "go together"),
        (dict(group_start=i32([0, 1, 2]), prefix_lens=i32([1]), prefix_pages=i32([[0]])),
         r"group_start is \[3\], expected \[2\]"),
    ]:
        with pytest.raises(L.OmgError, match=text):
            ops.PagedBatch(**{**good, **kw})


def test_validate():
    pool = torch.zeros((6, 16, 2, 1, 64), dtype=torch.float16)

    def batch(**kw):
        f = dict(q_start=[0, 1, 3], lens=[17, 2], pages=[[0, 1], [2, 9]], group_start=[0, 2],
                 prefix_lens=[20], prefix_pages=[[3, 4]])
        f.update(kw)
        return ops.PagedBatch(**{k: i32(v) for k, v in f.items()})

    batch().validate(pool, 3)
    for kw, text in [
        (dict(q_start=[0, 2, 1]), "q_start must ascend"),
        (dict(q_start=[0, 1, 4]), "q_start must ascend within 0..3"),
        (dict(lens=[33, 2]), "sequence 0 has 33 tokens in 2 pages"),
        (dict(lens=[17, 1]), "sequence 1 has 1 tokens, 2 of them new"),
        (dict(lens=[17, 17]), "sequence 1 uses page 9 of 6"),
        (dict(pages=[[0, -1], [2, 9]]), "sequence 0 uses page -1"),
        (dict(pages=[[0, 2], [2, 9]]), "append to one page"),
        (dict(group_start=[0, 1]), "group_start must ascend from 0 to 2"),
        (dict(prefix_lens=[40]), "prefix 0 has 40 tokens"),
        (dict(prefix_pages=[[3, 6]]), "prefix 0 uses page 6"),
    ]:
        with pytest.raises(L.OmgError, match=text):
            batch(**kw).validate(pool, 3)


def test_host_tensors_refused():
    pool = torch.zeros((6, 16, 2, 1, 64), dtype=torch.float16)
    b = ops.PagedBatch(i32([0, 1]), i32([1]), i32([[0]]))
    with pytest.raises(L.OmgError, match="on a GPU"):
        ops.paged_append(torch.zeros(1, 192), pool, b, heads=1)
    with pytest.raises(L.OmgError, match="on a GPU"):
        ops.paged_attention(torch.zeros(1, 1, 64, dtype=torch.float16), pool, b)
    with pytest.raises(L.OmgError, match="contiguous"):
        ops.paged_attention(torch.zeros(1, 1, 64, dtype=torch.float16), pool[:, ::2], b)
    with pytest.raises(L.OmgError, match="cache dtype"):
        ops.paged_append(torch.zeros(1, 192), pool.float(), b, heads=1)


def test_rope_frequencies():
    f = ops.rope_frequencies(1e6, 256, 64, scale=8.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,)
    assert np.allclose(f.numpy(), 1e6 ** (-np.arange(32) / 128) / 8, rtol=1e-15)
    for a in [(1e6, 256, 258), (1e6, 256, 3), (0.0, 256, 64)]:
        with pytest.raises(L.OmgError):
            ops.rope_frequencies(*a, device="cpu")


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "dtype 3"),
    (dict(rows=-1), "-1 rows"),
    (dict(vocab=0), "vocabulary of 0"),
    (dict(vocab=524289, stride=1 << 20), "vocabulary of 524289"),
    (dict(dtype=1, vocab=524289, stride=1 << 20), "vocabulary of 524289"),
    (dict(stride=99), "stride 99 < vocabulary 100"),
    (dict(logits=0), "logits is null"),
    (dict(logits=P + 2), "logits is not 4-byte aligned"),
    (dict(u=0), "u is null"),
    (dict(tokens=0), "tokens is null"),
])
def test_samples_refused(kw, text):
    f = dict(logits=P, stride=100, dtype=2, rows=2, vocab=100, u=P, temperature_all=1.0,
             top_p_all=1.0, tokens=P, probs=P)
    f.update(kw)
    refused(L.lib().omg_sample(0, C.byref(L.SampleArgsC(**f)), None), text)


def test_host_logits_refused():
    with pytest.raises(L.OmgError, match="on a GPU"):
        ops.sample(torch.zeros(1, 5), torch.zeros(1))

"""Host side of the 8-bit KV cache: record arithmetic and the refusals that come before any launch (no GPU needed)."""
import ctypes as C

import pytest
import torch

from pegaflow_b200 import _native as N
from tests import kv8_reference as ref

PTR = 0x10000    # never looked at: every call below is refused first


def cache(**kw):
    d = dict(data_ptr=PTR, block_stride_bytes=2064, kv_stride_bytes=2064 * 8, num_blocks=8, block_size=16, kv_heads=2, head_dim=64)
    d.update(kw)
    return N.Kv8CacheDesc(*[d[f] for f, _ in N.Kv8CacheDesc._fields_])


def batch(**kw):
    d = dict(block_tables=PTR, table_stride=4, max_blocks=4, n_seqs=2, lens=PTR, starts=PTR, status=None)
    d.update(kw)
    return N.Kv8Batch(*[d[f] for f, _ in N.Kv8Batch._fields_])


def attention(**kw):
    a = N.Kv8AttentionArgs(q=PTR, out=PTR, n_rows=2, max_query=1, q_row_stride=256, q_head_stride=64, out_row_stride=256,
                           out_head_stride=64, q_heads=4, dtype=0, causal=1, scale=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def evict(**kw):
    d = dict(weights=PTR, weights_seq_stride=64, weights_head_stride=32, weights_capacity=32, dst_tables=PTR + 64, dst_table_stride=2,
             keep=20, recent=4, new_lens=PTR, new_weights=PTR + 4096, new_capacity=32, kept=PTR)
    d.update(kw)
    return N.Kv8EvictArgs(*[d[f] for f, _ in N.Kv8EvictArgs._fields_])


def refused(status, word):
    assert status == 3 and word in N.lib.pf_last_error().decode(), (status, N.lib.pf_last_error())


@pytest.mark.parametrize("size,heads,dim,want", [(16, 8, 128, 16 * 8 * 128 + 32), (64, 1, 64, 64 * 64 + 16), (128, 5, 256, 128 * 5 * 256 + 32),
                                                 (16, 4, 64, 16 * 4 * 64 + 16), (48, 1, 64, 0), (16, 0, 64, 0), (16, 1, 96, 0),
                                                 (16, 1025, 64, 0), (8, 1, 64, 0), (0, 1, 64, 0)])
def test_record_bytes(size, heads, dim, want):
    assert N.lib.pf_kv8_record_bytes(size, heads, dim) == want


CACHES = [(dict(data_ptr=0), "null"), (dict(data_ptr=PTR + 8), "16 bytes"), (dict(block_stride_bytes=2072), "16 bytes"),
          (dict(block_stride_bytes=2048), "block stride"), (dict(kv_stride_bytes=1024), "K/V stride"), (dict(num_blocks=0), "num_blocks"),
          (dict(num_blocks=1 << 32), "num_blocks"), (dict(head_dim=80), "geometry"), (dict(block_size=24), "geometry")]
BATCHES = [(dict(block_tables=None), "null"), (dict(lens=None), "null"), (dict(max_blocks=0), "max_blocks"), (dict(max_blocks=1 << 24), "max_blocks"),
           (dict(n_seqs=8193), "limit")]


def every_call(c, b):
    c, b = C.byref(c) if c else None, C.byref(b) if b else None
    need = N.sz()
    yield N.lib.pf_kv8_append(0, c, b, PTR, PTR, 0, 2, 128, 64, 128, 64, None)
    yield N.lib.pf_kv8_attention_workspace(0, c, b, C.byref(attention()), C.byref(need))
    yield N.lib.pf_kv8_attention(0, c, b, C.byref(attention()), PTR, 1 << 40, None)
    yield N.lib.pf_kv8_evict(0, c, b, C.byref(evict()), None)


@pytest.mark.parametrize("bad,word", CACHES)
def test_every_call_refuses_a_bad_cache(bad, word):
    for status in every_call(cache(**bad), batch()):
        refused(status, word)


@pytest.mark.parametrize("bad,word", BATCHES)
def test_every_call_refuses_a_bad_batch(bad, word):
    for status in every_call(cache(), batch(**bad)):
        refused(status, word)


def test_null_structures():
    for status in every_call(None, batch()):
        refused(status, "null")
    for status in every_call(cache(), None):
        refused(status, "null")
    c, b = C.byref(cache()), C.byref(batch())
    refused(N.lib.pf_kv8_attention(0, c, b, None, PTR, 1, None), "null")
    refused(N.lib.pf_kv8_attention_workspace(0, c, b, C.byref(attention()), None), "null")
    refused(N.lib.pf_kv8_evict(0, c, b, None, None), "null")


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=2), "dtype"), (dict(n_rows=1 << 31), "2^31"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(k=PTR + 1), "aligned"),
    (dict(starts=None, n_rows=3), "evenly")])
def test_append_refusals(kw, word):
    d = dict(k=PTR, v=PTR, dtype=0, n_rows=2, starts=PTR)
    d.update(kw)
    refused(N.lib.pf_kv8_append(0, C.byref(cache()), C.byref(batch(starts=d["starts"])), d["k"], d["v"], d["dtype"], d["n_rows"],
                                128, 64, 128, 64, None), word)


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(q=PTR + 1), "aligned"), (dict(q_heads=3), "multiple"), (dict(q_heads=0), "multiple"),
    (dict(dtype=7), "dtype"), (dict(max_query=0), "max_query"), (dict(n_rows=1 << 31), "2^31"),
    (dict(n_rows=1 << 30, max_query=1 << 30), "too many query rows")])
def test_attention_refusals(kw, word):
    refused(N.lib.pf_kv8_attention(0, C.byref(cache()), C.byref(batch()), C.byref(attention(**kw)), PTR, 1 << 40, None), word)


def test_attention_refuses_rows_that_max_query_does_not_cover():
    refused(N.lib.pf_kv8_attention(0, C.byref(cache()), C.byref(batch(starts=None)), C.byref(attention(n_rows=4, max_query=1)), PTR,
                                   1 << 40, None), "max_query")


@pytest.mark.parametrize("kw,word", [
    (dict(keep=0), "keep"), (dict(recent=21), "recent"), (dict(new_capacity=19), "new_capacity"), (dict(weights=None), "null"),
    (dict(kept=None), "null"), (dict(new_weights=PTR), "weights"), (dict(dst_tables=PTR), "source"), (dict(dst_tables=None), "null"),
    (dict(new_lens=None), "null"), (dict(keep=1 << 31, new_capacity=1 << 31), "keep")])
def test_evict_refusals(kw, word):
    refused(N.lib.pf_kv8_evict(0, C.byref(cache()), C.byref(batch()), C.byref(evict(**kw)), None), word)


def test_the_python_class_needs_a_gpu_tensor():
    import pegaflow_b200 as pf

    with pytest.raises(ValueError, match="not on a GPU"):
        pf.Kv8Cache.from_tensor(torch.zeros((2, 4, 2064), dtype=torch.uint8), 16, 2, 64)
    with pytest.raises(ValueError, match="geometry"):
        pf.Kv8Cache.record_bytes(16, 2, 100)
    with pytest.raises(AttributeError):
        pf.NoSuchName


def test_a_calls_on_a_missing_device_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    assert N.lib.pf_kv8_append(0, C.byref(cache()), C.byref(batch()), PTR, PTR, 0, 2, 128, 64, 128, 64, None) == 4


def test_the_restatement_rounds_like_torch():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(20000, generator=g) * torch.exp2(torch.randint(-12, 6, (20000,), generator=g).float())
    x = x.clamp(-448, 448)
    assert torch.equal(ref.to_e4m3(x.double()), x.to(torch.float8_e4m3fn).double())
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[~torch.isnan(every)]
    assert torch.equal(ref.to_e4m3(every), every)
    for top in (448.0, 448.0001, 224.0, 1e-40, 3e38, 0.0, 449.0, 447.0, 2.0 ** -102 * 448):
        e = ref.exponent(top)
        assert top <= 448 * 2.0 ** e or e == ref.MAX_EXP
        assert e == ref.MIN_EXP or top > 448 * 2.0 ** (e - 1)


def test_eviction_order_of_the_restatement():
    nan = float("nan")
    assert ref.choose([1, 5, 5, 2, 9], 5, 3, 1) == [1, 2, 4]
    assert ref.choose([5, 5, 5, 5], 4, 2, 0) == [0, 1]
    assert ref.choose([nan, -1e30, nan, 0], 4, 3, 1) == [0, 1, 3]
    assert ref.choose([1, 2], 2, 5, 0) == [0, 1] and ref.choose([], 0, 5, 2) == []

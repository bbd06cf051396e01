"""Host side of the 8-bit KV cache at the edges: registration of caches in slices, refusals (no GPU needed)."""
import ctypes as C

import pytest
import torch

from pegaflow_b200 import _native as N
from tests.test_kv8_host import PTR, attention, batch, cache, evict, refused


class _Sliced:
    """What a Kv8Cache in a slice says of itself."""

    def registration(self):
        return (0x70000, 8 * 6192 * 2 - 2064), 8, 2064, 8 * 6192, 6192


def _worker(client):
    from pegaflow_b200.connector import PegaWorkerConnector

    return PegaWorkerConnector(client, None, instance_id="i", namespace="n", device_id=0, block_size=16)


def test_a_cache_in_a_slice_registers_its_records_and_their_stride():
    import pegaflow_b200 as pf

    seen = {}

    class Client(pf.InProcEngineClient):
        def __init__(self):
            pass

        def register_context_batch(self, *a, **kw):
            seen["args"], seen["kw"] = a, kw
            return True, ""

    w = _worker(Client())
    w.register_kv_caches({"a": _Sliced(), "b": torch.zeros((2, 8, 100), dtype=torch.uint8), "c": torch.zeros((8, 100), dtype=torch.uint8),
                          "d": torch.zeros((2, 1, 100), dtype=torch.uint8)})
    _, tensors, blocks, per_block, kv, segments = seen["args"][7:13]
    assert tensors[0] == (0x70000, 8 * 6192 * 2 - 2064) and blocks == [8, 8, 8, 1]
    assert per_block == [2064, 100, 100, 100] and kv == [8 * 6192, 800, 0, 100] and segments == [2, 2, 1, 2]
    assert seen["kw"] == {"block_stride_bytes_list": [6192, 100, 100, 200]}     # the others': what an engine takes by itself
    assert w.registrations["a"].bytes_per_block == 2064
    w.register_kv_caches({"b": torch.zeros((2, 8, 100), dtype=torch.uint8)})
    assert seen["kw"] == {}


def test_a_cache_in_a_slice_does_not_register_over_a_wire():
    class Client:
        def register_context_batch(self, *a, **kw):
            raise AssertionError("must not be called")

    with pytest.raises(ValueError, match="this process only"):
        _worker(Client()).register_kv_caches({"a": _Sliced()})


def test_clear_tail_is_one_of_its_values():
    for bad in (-1, 3):
        refused(N.lib.pf_kv8_attention(0, C.byref(cache()), C.byref(batch()), C.byref(attention(clear_tail=bad)), PTR, 1 << 40, None), "clear_tail")


def test_rows_are_not_divided_among_no_sequences():
    c, none = C.byref(cache()), C.byref(batch(n_seqs=0, starts=None))
    need = N.sz()
    refused(N.lib.pf_kv8_append(0, c, none, PTR, PTR, 0, 2, 128, 64, 128, 64, None), "evenly among 0")
    refused(N.lib.pf_kv8_attention_workspace(0, c, none, C.byref(attention()), C.byref(need)), "evenly among 0")
    refused(N.lib.pf_kv8_attention(0, c, none, C.byref(attention(clear_tail=1)), PTR, 1 << 40, None), "evenly among 0")
    assert N.lib.pf_kv8_append(0, c, none, None, None, 0, 0, 128, 64, 128, 64, None) == 0        # no rows: nothing to do
    assert N.lib.pf_kv8_append(0, c, C.byref(batch(n_seqs=0)), PTR, PTR, 0, 2, 128, 64, 128, 64, None) == 0
    assert N.lib.pf_kv8_evict(0, c, none, C.byref(evict()), None) == 0


def test_more_row_tiles_than_can_be_numbered_are_refused():
    rows = 1 << 24
    a = attention(n_rows=rows, max_query=rows)
    c, b = cache(), batch(n_seqs=8192)
    refused(N.lib.pf_kv8_attention(0, C.byref(c), C.byref(b), C.byref(a), PTR, 1 << 40, None), "too many query rows")


@pytest.mark.parametrize("rows,q_heads,max_blocks,fits", [(8 * 10240, 128, 8192, True), (8 * 10240, 128, 1 << 20, False), (8, 128, 1 << 20, True)])
def test_work_is_counted_in_the_tiles_that_the_rows_go_in(rows, q_heads, max_blocks, fits):
    """8 prompts of 10240 rows, 128 query and 8 KV heads: tables for 131072 tokens are 80 tiles of 256 rows x 1029 units of a head,
    not 20480 of 4 rows.  Where there is no device the call ends behind its checks, with that error."""
    need = N.sz()
    c = cache(kv_heads=8, head_dim=128, block_stride_bytes=16 * 8 * 128 + 32, kv_stride_bytes=8 * (16 * 8 * 128 + 32))
    a = attention(n_rows=rows, max_query=rows // 8, q_heads=q_heads)
    status = N.lib.pf_kv8_attention_workspace(0, C.byref(c), C.byref(batch(n_seqs=8, max_blocks=max_blocks)), C.byref(a), C.byref(need))
    if fits:
        assert status == (0 if torch.cuda.is_available() else 4)
    else:
        refused(status, "too many query rows")


CLEAN = dict(n_rows=4, max_query=2, q_heads=4, q=PTR, out=PTR + (1 << 20), q_row_stride=256, q_head_stride=64, out_row_stride=256, out_head_stride=64)


def attended(**kw):
    d = dict(CLEAN, **kw)
    return N.lib.pf_kv8_attention(0, C.byref(cache()), C.byref(batch(starts=None)), C.byref(attention(**d)), None, 0, None)


@pytest.mark.parametrize("kw,word", [
    (dict(out_row_stride=0), "out"), (dict(out_head_stride=0), "out"), (dict(out_row_stride=255), "out"), (dict(out_head_stride=63), "out"),
    (dict(out_row_stride=64, out_head_stride=255), "out"), (dict(out_row_stride=64, out_head_stride=64), "out"),
    (dict(weights=PTR, weights_seq_stride=0, weights_head_stride=32, weights_capacity=32), "weights"),
    (dict(weights=PTR, weights_seq_stride=64, weights_head_stride=31, weights_capacity=32), "weights"),
    (dict(out=PTR + 128), "q"), (dict(out=PTR + 2), "q"), (dict(out=PTR - 512), "q"), (dict(out=PTR, out_row_stride=512), "q"),
    (dict(q_row_stride=512, out_row_stride=512, out=PTR + 2 * 256 - 2), "q"), (dict(q_row_stride=512, out_row_stride=512, out=PTR + 2 * 256 + 1), "aligned")])
def test_outputs_that_overlap_are_refused(kw, word):
    refused(attended(**kw), word)


@pytest.mark.parametrize("kw", [
    {}, dict(out=PTR), dict(out_row_stride=64, out_head_stride=256),                       # apart, in place, heads outermost
    dict(q_row_stride=512, out_row_stride=512, out=PTR + 2 * 256), dict(q_row_stride=512, out_row_stride=512, out=PTR - 2 * 256),   # rows in turn
    dict(q_row_stride=512, q_head_stride=128, out_row_stride=512, out_head_stride=128, out=PTR + 128),                          # heads in turn
    dict(n_rows=2, max_query=1, q_heads=2, out_row_stride=192, out_head_stride=64),
    dict(weights=PTR, weights_seq_stride=64, weights_head_stride=32, weights_capacity=32),
    dict(weights=PTR, weights_seq_stride=32, weights_head_stride=64, weights_capacity=32)])
def test_outputs_that_do_not_overlap_get_past_the_checks(kw):
    """What comes next is the device, or (where there is one) the workspace that this call does not have."""
    status = attended(**kw)
    assert status == 4 or (status == 3 and b"workspace" in N.lib.pf_last_error()), (status, N.lib.pf_last_error())


def test_the_overlap_checks_agree_with_a_search_of_all_elements():
    """Small random layouts: whatever shares an element is refused, but for q itself; most of what does not is let through."""
    g = torch.Generator().manual_seed(3)
    among = lambda x: x[int(torch.randint(0, len(x), (1,), generator=g))]  # noqa: E731
    steps = [0, 32, 64, 96, 128, 160, 192, 256, 288, 384]
    seen = {True: 0, False: 0}
    for _ in range(800):
        rows, heads, delta = among([2, 4]), among([2, 4]), 32 * among(range(-24, 25))
        q_strides, strides = (among(steps), among(steps)), (among(steps), among(steps))
        if among([True, False]):
            strides = q_strides
        status = attended(n_rows=rows, max_query=rows // 2, q_heads=heads, out=PTR + 2 * delta, q_row_stride=q_strides[0], q_head_stride=q_strides[1],
                          out_row_stride=strides[0], out_head_stride=strides[1])
        told = status == 3 and b"overlap" in N.lib.pf_last_error()
        places = lambda at, s: [at + i * s[0] + j * s[1] + d for i in range(rows) for j in range(heads) for d in range(64)]  # noqa: E731
        q, out = places(0, q_strides), places(delta, strides)
        shared = len(set(out)) < len(out) or (not set(q).isdisjoint(out) and not (delta == 0 and strides == q_strides))
        assert told or not shared, (rows, heads, delta, q_strides, strides)
        if not shared:
            seen[told] += 1
    assert seen[False] > 2 * seen[True]


def test_eviction_into_rows_that_overlap_is_refused():
    for stride in (0, 1):
        refused(N.lib.pf_kv8_evict(0, C.byref(cache()), C.byref(batch()), C.byref(evict(dst_table_stride=stride)), None), "overlap")
    assert N.lib.pf_kv8_evict(0, C.byref(cache()), C.byref(batch(n_seqs=0)), C.byref(evict(dst_table_stride=0)), None) == 0

"""The 8-bit KV cache on a GPU at the edges of what its calls allow: pages that are missing, rows of no sequence, tensors
of other streams, caches in slices of a buffer, sizes beyond the other tests'."""
import math

import pytest
import torch

from tests import kv8_reference as ref
from tests.test_gpu_kv8 import bytes_of, gen, ints, make_cache, make_tables, pf, same_bytes, starts_of  # noqa: F401

pytestmark = pytest.mark.gpu


def rows_of(cache, kv, table, n):
    """float64 [kv_heads, n, dim] on the GPU: what the first n tokens of a block table hold; 0 for pages that are not there."""
    size = cache.block_size
    ids = torch.tensor(table[: -(-n // size)], dtype=torch.long, device="cuda")
    there = (ids >= 0) & (ids < cache.num_blocks)
    at = torch.where(there, ids, torch.zeros_like(ids))
    x = cache.values[kv, at].double() * cache.scales[kv, at].double()[:, :, None, None]
    x = torch.where(there[:, None, None, None], x, torch.zeros_like(x))
    return x.transpose(0, 1).reshape(cache.kv_heads, -1, cache.head_dim)[:, :n], there.repeat_interleave(size)[:n]


def plain(cache, q, table, n, scale, causal=True):
    """64 bits, one sequence: (out, lse, weights, sum p |v|, spread); a row that sees nothing gives 0, -infinity and no weight."""
    rows, q_heads, dim = q.shape
    heads, group = cache.kv_heads, q_heads // cache.kv_heads
    (k, there), (v, _) = rows_of(cache, 0, table, n), rows_of(cache, 1, table, n)
    last = n - rows + torch.arange(rows, device="cuda") if causal else torch.full((rows,), n, device="cuda")
    see = (torch.arange(n, device="cuda")[None] <= last[:, None]) & there
    x = torch.einsum("ihgd,hjd->ihgj", q.double().view(rows, heads, group, dim), k) * scale
    x = x.masked_fill(~see[:, None, None], -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.where(torch.isneginf(lse)[..., None], torch.zeros_like(x), torch.exp(x - lse[..., None]))
    spread = (torch.einsum("ihgd,hjd->ihgj", q.double().abs().view(rows, heads, group, dim), k.abs()) * abs(scale) * see[:, None, None]).amax(-1)
    back = lambda t: t.reshape(rows, q_heads, dim)  # noqa: E731
    return (back(torch.einsum("ihgj,hjd->ihgd", p, v)), lse.reshape(rows, q_heads), p.sum((0, 2)),
            back(torch.einsum("ihgj,hjd->ihgd", p, v.abs())), spread.reshape(rows, q_heads))


def close(cache, q, got, lse, weights, before, want, n):
    """The bounds of tests/test_gpu_kv8.py: ds of a score, p to 2^-21 and, for the product with V, 2^-11, sums of n terms."""
    out, want_lse, w, size, spread = want
    dim, rows = q.shape[2], q.shape[0] * q.shape[1] // cache.kv_heads
    ds = (dim + 8) * 2.0 ** -23 * spread
    rel = 2 * (ds + 2.0 ** -21) + 2.0 ** -11 + 2 * n * 2.0 ** -24
    big = float((cache.values.double().abs().nan_to_num() * cache.scales.double()[..., None, None]).max())
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    tol = size * rel[..., None] + half * out.abs() + big * n * (2.0 ** -27 if rows <= 32 else 2.0 ** -30) + 1e-30
    assert ((got.double() - out).abs() <= tol).all()
    if lse is not None:
        none = torch.isneginf(want_lse)
        assert torch.equal(torch.isneginf(lse.double()), none)
        assert ((lse.double() - want_lse).abs() <= 2 * ds + 2.0 ** -20 + 2.0 ** -22 * want_lse.abs() + n * 2.0 ** -24)[~none].all()
    if weights is not None:
        # score and lse are off by ds each, twice where they are computed twice; rows terms are added, then one more
        worst = 4 * float(ds.max()) + 2.0 ** -19 + n * 2.0 ** -23 + rows * 2.0 ** -24
        total = before.double() + w
        assert ((weights.double() - total).abs() <= w * worst + 2.0 ** -23 * total).all()


# ------------------------------------------------------------------------------------------------ pages that are missing
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 2, 5, 40])
@pytest.mark.parametrize("missing", ["first", "all", "from the fourth on"])
def test_weights_of_rows_that_see_missing_pages_only(pf, dim, rows, missing):
    """One row or several row tiles, scores kept or taken again: rows of which every visible page is missing weigh nothing, and
    tokens that other rows see get those rows' weights."""
    size, heads, group, n = 16, 2, 4, 16 + rows - 1 if missing == "first" else 90      # row 0 sees the first page alone
    blocks, tables = make_tables([n], size, 201)
    cache = make_cache(pf, blocks, size, heads, dim, 202)
    table = tables[0].tolist()
    gone = {"first": [0], "all": range(len(table)), "from the fourth on": range(3, len(table))}[missing]
    for i in gone:
        table[i] = -1 if i % 2 else blocks
    q = torch.randn((rows, heads * group, dim), generator=gen(203), device="cuda").bfloat16()
    w = torch.rand((1, heads, n + 3), generator=gen(204), device="cuda")
    before = w.clone()
    out, lse = cache.attention(q, ints([table]), ints([n]), weights=w, lse=True)
    with pytest.raises(pf.PegaflowInvalidArgument, match="block id"):
        cache.check()
    assert torch.isfinite(w).all() and torch.equal(w[..., n:], before[..., n:])
    close(cache, q, out, lse, w[0, :, :n], before[0, :, :n], plain(cache, q, table, n, dim ** -0.5), n)


# ------------------------------------------------------------------------------------------------ caches in slices of a buffer
SLICES = {
    # shape of the buffer (2: K and V, 12 blocks, 3 layers), a layer's cache in it
    "layers within a block": (lambda r: (2, 12, 3, r), lambda t, i: t[:, :, i]),
    "layers outermost": (lambda r: (3, 2, 12, r), lambda t, i: t[i]),
    "K and V of a block together": (lambda r: (12, 3, 2, r), lambda t, i: t[:, i].transpose(0, 1)),
    "records with room behind them": (lambda r: (2, 12, 3, r + 48), lambda t, i: t[:, :, i]),
}


@pytest.mark.parametrize("only", [None, 0])
@pytest.mark.parametrize("layout", SLICES)
def test_caches_in_a_slice_of_a_larger_buffer_are_saved_and_loaded_alone(pf, layout, only):
    """A load writes the records of its own layer, block and all, and leaves every other byte of the buffer as it was; so
    does a peer copy."""
    from pegaflow_b200 import connector

    size, heads, dim = 16, 2, 64
    shape, slice_of = SLICES[layout]
    record = pf.Kv8Cache.record_bytes(size, heads, dim)
    buffers = [torch.randint(0, 256, shape(record), dtype=torch.uint8, device="cuda", generator=gen(210 + i)) for i in range(2)]
    use = [0, 1, 2] if only is None else [only]
    caches = [{f"l{i}": pf.Kv8Cache.from_tensor(slice_of(b, i), size, heads, dim) for i in use} for b in buffers]
    eng = pf.PegaEngine(64 << 20)
    client = connector.InProcEngineClient(eng)
    conns = [connector.PegaWorkerConnector(client, eng, instance_id=who, namespace="kv8", device_id=0, block_size=size) for who in "ab"]
    for conn, c in zip(conns, caches):
        conn.register_kv_caches(c)
        assert all(conn.registrations[n].bytes_per_block == record for n in c)
    src, home = [2, 7, 11], [5, 1, 9]
    hashes = [b"slice-%d" % i for i in range(3)]
    torch.cuda.synchronize()
    conns[0].wait_for_save([(n, src, hashes) for n in caches[0]])
    want = buffers[1].clone()
    for i in use:
        slice_of(want, i)[:, home, :record] = slice_of(buffers[0], i)[:, src, :record]
    hit = client.query_prefetch("b", hashes, "r")
    assert hit.num_hit_blocks == 3
    torch.cuda.synchronize()
    conns[1].start_load_kv([("r", hit.lease, home)])
    done = []
    while not done:
        done, failed = conns[1].get_finished()
        assert not failed
    torch.cuda.synchronize()
    assert torch.equal(buffers[1], want)
    eng.peer_load("a", 0, "b", 0, src, [4, 3, 0])
    for i in use:
        slice_of(want, i)[:, [4, 3, 0], :record] = slice_of(buffers[0], i)[:, src, :record]
    torch.cuda.synchronize()
    assert torch.equal(buffers[1], want)
    for conn in conns:
        conn.unregister()
    eng.close()


# ------------------------------------------------------------------------------------------------ rows of no sequence
def leave_behind(*shapes):
    """Fills memory that the allocator gives out next for tensors of these shapes and types, and returns it."""
    torch.cuda.synchronize()
    for shape, dtype in shapes:
        keep = [torch.full(shape, 7.0, dtype=dtype, device="cuda") for _ in range(64)]
        del keep
    torch.cuda.synchronize()


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("before,counts,behind", [(3, [1, 1], 0), (0, [1, 1], 3), (2, [3, 0, 2], 2), (5, [], 0), (4, [0, 0], 1), (1, [40, 3], 2)])
def test_rows_in_front_of_and_behind_the_sequences(pf, before, counts, behind, given):
    """0 and -infinity where the call allocates the output, left as they were in a given one; lse is the call's own always."""
    n_seqs, rows = len(counts), before + sum(counts) + behind
    lens = [70, 33, 50][:n_seqs]
    blocks, tables = make_tables(lens, 16, 220) if n_seqs else (4, torch.zeros((0, 2), dtype=torch.int32))
    cache = make_cache(pf, blocks, 16, 2, 64, 221)
    q = torch.randn((rows, 8, 64), generator=gen(222), device="cuda").half()
    none = torch.ones(rows, dtype=torch.bool, device="cuda")
    none[before:before + sum(counts)] = False
    q[none] = math.nan
    starts = [before + n for n in starts_of(counts)]
    out = torch.full_like(q, 3.0) if given else None
    leave_behind((q.shape, q.dtype), ((rows, 8), torch.float32))
    got, lse = cache.attention(q, tables.cuda(), ints(lens), starts=ints(starts), max_query=max([1] + counts), lse=True, out=out)
    cache.check()
    assert (got[none] == (3.0 if given else 0.0)).all() and torch.isneginf(lse[none]).all()
    for s, n in enumerate(counts):
        if n:
            a = slice(starts[s], starts[s] + n)
            close(cache, q[a], got[a], lse[a], None, None, plain(cache, q[a], tables[s].tolist(), lens[s], 0.125), lens[s])


def test_append_takes_the_rows_behind_its_first_start(pf):
    """Rows in front of starts[0], a batch's other part, are not read: their NaN reach nothing."""
    cache, same = make_cache(pf, 6, 16, 2, 64, 223), make_cache(pf, 6, 16, 2, 64, 223)
    x = torch.randn((9, 2, 64), generator=gen(224), device="cuda").half()
    x[:4] = math.nan
    cache.append(x, -x, ints([[1], [4]]), ints([3, 0]), starts=ints([4, 6, 9]))
    same.append(x[4:], -x[4:], ints([[1], [4]]), ints([3, 0]), starts=ints([0, 2, 5]))
    cache.check()
    assert torch.equal(cache.tensor, same.tensor)


def test_rows_without_a_sequence_are_refused(pf):
    """Rows cannot be divided among no sequences; with starts they are rows of no sequence."""
    cache = pf.Kv8Cache(4, 16, 2, 64)
    x = torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    none, nothing = torch.zeros((0, 2), dtype=torch.int32, device="cuda"), ints([])
    for call in (lambda: cache.attention(x, none, nothing), lambda: cache.attention(x, none, nothing, lse=True, out=torch.empty_like(x)),
                 lambda: cache.append(x, x, none, nothing)):
        with pytest.raises(pf.PegaflowInvalidArgument, match="evenly"):
            call()
    assert cache.attention(x[:0], none, nothing).shape == (0, 2, 64)
    cache.append(x[:0], x[:0], none, nothing)
    cache.append(x, x, none, nothing, starts=ints([0]))
    cache.check()
    assert (cache.tensor == 0).all()


# ------------------------------------------------------------------------------------------------ sizes
@pytest.mark.parametrize("seqs,n,width,heads", [(64, 512, 64, 2), (8192, 4096, 8192, 64)])
def test_row_starts_that_fall_again_and_again_do_no_harm(pf, seqs, n, width, heads):
    """Starts 0, n, 0, n, ... claim all rows for every second sequence, more work than these rows can be (in the second
    case more than 32 bits count): no row is computed, and the call says why."""
    cache = make_cache(pf, 8, 16, heads, 64, 260)
    q = torch.randn((n, 8 * heads, 64), generator=gen(261), device="cuda").half()
    tables = ints([[1, 2]]).repeat(1, width // 2).expand(seqs, width)
    lens = torch.full((seqs,), 16 * width, dtype=torch.int32, device="cuda")
    starts = ints([0, n] * (seqs // 2) + [0])
    out, lse = cache.attention(q, tables, lens, starts=starts, max_query=n, causal=False, lse=True)
    with pytest.raises(pf.PegaflowInvalidArgument, match="row starts"):
        cache.check()
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_row_starts_that_fall_again_and_again_leave_weights_as_they_are(pf, dim):
    """Without an lse of the call's own; a given out stays too."""
    size, heads, seqs, rows = 16, 2, 400, 200
    cache = make_cache(pf, 8, size, heads, dim, 267)
    q = torch.randn((rows, 4 * heads, dim), generator=gen(268), device="cuda").half()
    tables, lens = ints([[1, 2, 3, 4]]).expand(seqs, 4), torch.full((seqs,), 64, dtype=torch.int32, device="cuda")
    w = torch.rand((seqs, heads, 64), generator=gen(269), device="cuda")
    before, out = w.clone(), torch.full_like(q, 3.0)
    cache.attention(q, tables, lens, starts=ints([0, rows] * (seqs // 2) + [0]), max_query=rows, weights=w, out=out)
    with pytest.raises(pf.PegaflowInvalidArgument, match="row starts"):
        cache.check()
    assert torch.equal(w, before) and (out == 3).all()


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_a_row_start_that_falls_behind_the_sequences_cuts_those_rows_alone(pf, rows):
    """A batch padded with sequences whose starts are 0: reported, and the others' rows are computed as ever."""
    size, heads, dim, n = 16, 2, 128, 100
    blocks, tables = make_tables([n, n - 10], size, 266)
    cache = make_cache(pf, blocks, size, heads, dim, 267)
    q = torch.randn((2 * rows + 3, 4 * heads, dim), generator=gen(268), device="cuda").half()
    t = torch.cat([tables, torch.zeros((2, tables.shape[1]), dtype=torch.int32)]).cuda()
    w = torch.rand((4, heads, n), generator=gen(269), device="cuda")
    before = w.clone()
    out, lse = cache.attention(q, t, ints([n, n - 10, 0, 0]), starts=ints([0, rows, 2 * rows, 0, 0]), max_query=rows, weights=w, lse=True)
    with pytest.raises(pf.PegaflowInvalidArgument, match="row starts"):
        cache.check()
    for s in range(2):
        a, m = slice(s * rows, (s + 1) * rows), n - 10 * s
        close(cache, q[a], out[a], lse[a], w[s, :, :m], before[s, :, :m], plain(cache, q[a], tables[s].tolist(), m, dim ** -0.5), m)
    assert torch.equal(w[2:], before[2:])


def test_prompts_over_wide_tables_are_counted_by_their_own_tiles(pf):
    """8 prompts of 300 rows with tables for 2^24 tokens, of which they use 400."""
    size, heads, group, dim, rows = 16, 2, 16, 64, 300
    lens = [400] * 8
    blocks, tables = make_tables(lens, size, 265, width=1 << 20)
    cache = make_cache(pf, blocks, size, heads, dim, 263)
    q = torch.randn((8 * rows, heads * group, dim), generator=gen(264), device="cuda").bfloat16()
    out, lse = cache.attention(q, tables.cuda(), ints(lens), lse=True)
    cache.check()
    for s in (0, 7):
        a = slice(s * rows, (s + 1) * rows)
        close(cache, q[a], out[a], lse[a], None, None, plain(cache, q[a], tables[s].tolist(), lens[s], 0.125), lens[s])


# ------------------------------------------------------------------------------------------------ streams
LONG = 200_000_000       # cycles, a tenth of a second: longer than the host takes for everything behind it


def operators(cache, x, t, n, w):
    """Each operator as a call with `stream`, on tensors that the call alone holds: temporaries of the current stream."""
    starts, dst = ints([0, 1, 2]), ints([[7], [8]])
    return {
        "append": lambda s: cache.append(x.half(), (-x).half(), t + 0, n + 0, starts=starts + 0, stream=s),
        "attention": lambda s: cache.attention(x.repeat(1, 2, 1).half(), t + 0, n + 0, starts=starts + 0, max_query=1, weights=w, lse=True, stream=s),
        "evict": lambda s: cache.evict(t + 0, n + 0, w + 0, dst + 0, 9, recent=2, stream=s),
    }


def overwrite():
    """What the allocator gives out next for tensors like the calls' is full of ones."""
    for like in ((2, 2, 64), (2, 4, 64), (2, 2, 30), (2, 2), (2,), (3,), (2, 1)):
        for dtype in (torch.float32, torch.float16, torch.int32):
            keep = [torch.full(like, 1, dtype=dtype, device="cuda") for _ in range(4)]
            del keep


@pytest.mark.parametrize("late", ["caller", "stream"])
@pytest.mark.parametrize("name", ["append", "attention", "evict"])
def test_a_given_stream_takes_temporaries_of_the_current_one(pf, name, late):
    """The work on `stream` comes behind what the current stream was given before the call, and the call's tensors are not
    given out again before it has read them: whichever of the two streams is far behind."""
    results = []
    for own_stream in (False, True):
        cache = make_cache(pf, 9, 16, 2, 64, 230)
        x = torch.randn((2, 2, 64), generator=gen(231), device="cuda")
        t, n, w = ints([[1, 2], [3, 4]]), ints([20, 17]), torch.rand((2, 2, 30), generator=gen(232), device="cuda")
        call = operators(cache, x, t, n, w)[name]
        side = torch.cuda.Stream()
        overwrite()
        torch.cuda.synchronize()
        if own_stream:
            with torch.cuda.stream(side if late == "stream" else torch.cuda.current_stream()):
                torch.cuda._sleep(LONG)
            got = call(side.cuda_stream)
            overwrite()
        else:
            got = call(None)
        torch.cuda.synchronize()
        cache.check()
        results.append((cache.tensor.clone(), w.clone(), got if isinstance(got, tuple) else ()))
    (a, wa, oa), (b, wb, ob) = results
    assert torch.equal(a, b) and torch.equal(wa, wb) and len(oa) == len(ob)
    assert all(torch.equal(p, q) for p, q in zip(oa, ob))


def test_outputs_made_on_a_given_stream_outlive_their_use_on_the_current_one(pf):
    """The current stream, which waits for the other one, still reads an output after its last name is gone."""
    cache = make_cache(pf, 9, 16, 2, 64, 233)
    q = torch.randn((2, 8, 64), generator=gen(234), device="cuda").half()
    t, n = ints([[1, 2], [3, 4]]), ints([20, 17])
    want = cache.attention(q, t, n)
    side = torch.cuda.Stream()

    def others():
        with torch.cuda.stream(side):
            keep = [torch.full(q.shape, 1, dtype=q.dtype, device="cuda") for _ in range(4)]
            del keep

    others()                                   # what is loaded at its first use waits for the whole device
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    got = cache.attention(q, t, n, stream=side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(LONG)
    copy = got.clone()
    del got
    others()
    torch.cuda.synchronize()
    assert torch.equal(copy, want)


def test_a_given_stream_joins_the_capture_of_the_current_one(pf):
    """Calls on another stream while the current one is captured: they become part of the graph, which the caller joins; a stream
    that is captured alone takes calls too."""
    cache = make_cache(pf, 9, 16, 2, 64, 240)
    q = torch.randn((2, 8, 64), generator=gen(241), device="cuda").half()
    t, n = ints([[1, 2], [3, 4]]), ints([20, 17])
    want = cache.attention(q, t, n)
    side, torch_graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(torch_graph):
        got = cache.attention(q + 0, t, n, stream=side.cuda_stream)
        torch.cuda.current_stream().wait_stream(side)
        got = got + 0
    alone = torch.cuda.CUDAGraph()
    capturing, current = torch.cuda.Stream(), torch.cuda.current_stream()
    out = torch.zeros_like(q)
    with torch.cuda.graph(alone, stream=capturing):
        with torch.cuda.stream(current):
            handle = capturing.cuda_stream
            cache.attention(q, t, n, out=out, stream=handle)
    for _ in range(2):
        torch_graph.replay()
        alone.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(out, want)
        got.zero_(), out.zero_()


def test_a_new_cache_is_ready_for_every_stream(pf):
    """Its zeros and its status are there when the constructor returns, however far behind the current stream is."""
    side = torch.cuda.Stream()
    x = torch.ones((1, 2, 64), dtype=torch.float16, device="cuda")
    t, n = ints([[9]]), ints([0])
    warm = pf.Kv8Cache(4, 16, 2, 64)
    del warm
    torch.cuda.synchronize()
    torch.cuda._sleep(LONG)
    cache = pf.Kv8Cache(4, 16, 2, 64)
    with torch.cuda.stream(side):
        cache.append(x, x, t, n)               # a block that is not there
    side.synchronize()
    torch.cuda.synchronize()
    with pytest.raises(pf.PegaflowInvalidArgument, match="block id"):
        cache.check()
    assert (cache.tensor == 0).all()


# ------------------------------------------------------------------------------------------------ refusals
def test_tangents_and_gradients_are_refused(pf):
    """There is neither a backward pass nor a forward-mode rule: nothing that carries a derivative is taken."""
    import torch.autograd.forward_ad as fwad

    cache = pf.Kv8Cache(6, 16, 2, 64)
    t, n, dst = ints([[1, 2]]), ints([20]), ints([[3]])
    x, w = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((1, 2, 32), device="cuda")
    calls = [lambda x, w: cache.append(x, torch.zeros_like(x), t, n), lambda x, w: cache.append(torch.zeros_like(x), x, t, n),
             lambda x, w: cache.attention(x, t, n), lambda x, w: cache.attention(torch.zeros_like(x), t, n, out=x),
             lambda x, w: cache.attention(torch.zeros_like(x), t, n, weights=w), lambda x, w: cache.evict(t, n, w, dst, 8)]
    uses_x = [True, True, True, True, False, False]
    for call, of_x in zip(calls, uses_x):
        with fwad.dual_level():
            a = fwad.make_dual(x.clone(), torch.ones_like(x)) if of_x else x.clone()
            b = w.clone() if of_x else fwad.make_dual(w.clone(), torch.ones_like(w))
            with pytest.raises(pf.PegaflowInvalidArgument, match="backward"):
                call(a, b)
        with pytest.raises(pf.PegaflowInvalidArgument, match="backward"):
            call(x.clone().requires_grad_() if of_x else x, w if of_x else w.clone().requires_grad_())
        with torch.no_grad():
            call(x.clone().requires_grad_() if of_x else x.clone(), w.clone() if of_x else w.clone().requires_grad_())
    with fwad.dual_level():
        cache.attention(x, t, n, weights=w)          # nothing here carries a tangent
    cache.check()


def test_outputs_that_overlap_themselves_or_the_queries_are_refused(pf):
    """Several CTAs would write one element, or one would read what another has written."""
    cache = pf.Kv8Cache(6, 16, 2, 64)
    t, n = ints([[1, 2], [3, 4]]), ints([20, 7])
    q = torch.randn((2, 4, 64), generator=gen(250), device="cuda").half()
    w = torch.zeros((2, 2, 32), device="cuda")
    many = q.repeat(20, 1, 1)               # 40 rows of a KV head: their weights take the queries a second time
    buffer = torch.zeros(4096, dtype=torch.float16, device="cuda")
    E = pf.PegaflowInvalidArgument
    for bad in (lambda: cache.attention(q, t, n, out=q.new_zeros((1, 4, 64)).expand(2, 4, 64)),
                lambda: cache.attention(q, t, n, out=q.new_zeros((2, 1, 64)).expand(2, 4, 64)),
                lambda: cache.attention(q, t, n, out=buffer.as_strided((2, 4, 64), (200, 64, 1))),
                lambda: cache.attention(q, t, n, weights=w[:1].expand(2, 2, 32)), lambda: cache.attention(q, t, n, weights=w[:, :1].expand(2, 2, 32)),
                lambda: cache.evict(t, n, w, ints([[5]]).expand(2, 1), 8),
                lambda: cache.attention(buffer[:512].view(2, 4, 64), t, n, out=buffer[64:576].view(2, 4, 64)),
                lambda: cache.attention(many, t, n, out=many, weights=w)):
        with pytest.raises(E, match="overlap"):
            bad()
    cache.check()
    # in place, and between the queries: as before
    want = cache.attention(q, t, n)
    fused = torch.zeros((2, 12, 64), dtype=torch.float16, device="cuda")
    fused[:, 4:8] = q
    cache.attention(fused[:, 4:8], t, n, out=fused[:, :4])
    assert torch.equal(fused[:, :4], want) and torch.equal(fused[:, 4:8], q) and (fused[:, 8:] == 0).all()
    apart = torch.zeros((2, 4, 2, 64), dtype=torch.float16, device="cuda")
    apart[:, :, 1] = q
    cache.attention(apart[:, :, 1], t, n, out=apart[:, :, 0])
    assert torch.equal(apart[:, :, 0], want)
    mine = q.clone()
    assert torch.equal(cache.attention(mine, t, n, out=mine), want)
    mine = q.clone()
    assert torch.equal(cache.attention(mine, t, n, out=mine, weights=w), want)
    mine = many.clone()
    assert torch.equal(cache.attention(mine, t, n, out=mine), cache.attention(many, t, n))
    one = cache.attention(q[:1], t[:1], n[:1], out=q.new_zeros((1, 4, 64)).expand(1, 4, 64))      # of one row any stride
    assert torch.equal(one, want[:1])


def test_all_three_in_one_graph_with_a_given_stream(pf):
    """A step of append, attention and eviction captured together, on the capturing stream by name; replayed with other
    lengths and rows, it gives what the calls give."""
    size, heads, dim = 16, 2, 64
    cache, same = make_cache(pf, 12, size, heads, dim, 235), make_cache(pf, 12, size, heads, dim, 235)
    t, dst = ints([[1, 2, 3], [4, 5, 6]]), ints([[7], [8]])
    x = torch.randn((2, heads, dim), generator=gen(236), device="cuda").half()
    q = torch.randn((2, 2 * heads, dim), generator=gen(237), device="cuda").half()
    lens, w = ints([20, 31]), torch.zeros((2, heads, 48), device="cuda")

    def step(c, stream):
        c.append(x, -x, t, lens, stream=stream)
        out = c.attention(q, t, lens + 1, weights=w, stream=stream)
        return (out, *c.evict(t, lens + 1, w, dst, 10, recent=3, stream=stream))

    step(cache, None)
    torch.cuda.synchronize()
    cache.tensor.copy_(same.tensor)
    graph, capturing = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=capturing):
        got = step(cache, capturing.cuda_stream)
    for lengths in ([20, 31], [0, 47], [15, 16]):
        lens.copy_(ints(lengths))
        x.copy_(torch.randn((2, heads, dim), generator=gen(238 + lengths[0]), device="cuda"))
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        weights = w.clone()
        w.zero_()
        want = step(same, None)
        assert torch.equal(weights, w) and all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(cache.tensor, same.tensor)
    cache.check()


@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
@pytest.mark.parametrize("lens,keep,recent", [([12288, 12289, 40], 7000, 33), ([30001], 12300, 0), ([20000, 12287], 19999, 5000)])
def test_evict_from_rows_longer_than_the_choice_holds_in_registers(pf, lens, keep, recent, kind):
    size, heads, dim = 64, 1, 64
    blocks, tables = make_tables(lens, size, 270)
    n_dst = -(-keep // size)
    cache = make_cache(pf, blocks + len(lens) * n_dst, size, heads, dim, 271, wide=5)
    dst = torch.arange(blocks, blocks + len(lens) * n_dst, dtype=torch.int32).view(len(lens), n_dst)
    w = torch.exp(2 * torch.randn((len(lens), heads, max(lens)), generator=gen(272), device="cuda"))
    if kind == "ties":
        w = torch.floor(w)
    elif kind == "special":
        w[..., ::3] = 0
        w[..., 1::7] = math.nan
        w[..., 2::11] = math.inf
        w[..., 4::13] = -0.0
    before, old, want = bytes_of(cache), ref.Cache(cache), ref.Cache(cache)
    new_lens, new_w, kept = cache.evict(tables.cuda(), ints(lens), w, dst.cuda(), keep, recent=recent)
    cache.check()
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    w_ = w.cpu()
    for s, n in enumerate(lens):
        at = ref.choose(w_[s, 0].tolist(), n, keep, recent)
        assert kept[s, 0].tolist() == at + [-1] * (keep - len(at))
        want_w = torch.zeros(new_w.shape[2])
        want_w[: len(at)] = w_[s, 0, at]
        assert torch.equal(new_w[s, 0].cpu().nan_to_num(-7.0), want_w.nan_to_num(-7.0))
        ids = tables[s].long()
        for kv in range(2):
            x = (old.values[kv, ids, 0] * old.scales[kv, ids, 0][:, None, None]).reshape(-1, dim)[at]
            for b in range(-(-len(at) // size)):
                want.store(kv, int(dst[s, b]), 0, {i: x[b * size + i] for i in range(min(size, len(at) - b * size))})
    same_bytes(cache, want, before)


@pytest.mark.parametrize("dim", [64, 128])
def test_weights_of_several_row_tiles_over_ranges_longer_than_a_pass(pf, dim):
    """Eight requests whose tokens give each CTA more steps than it sums the weights of at a time."""
    size, heads, group, rows, lens = 64, 8, 4, 20, [10240, 9000, 10240, 8111, 10240, 10001, 10240, 10240]
    blocks, tables = make_tables(lens, size, 280)
    cache = make_cache(pf, blocks, size, heads, dim, 281)
    q = torch.randn((8 * rows, heads * group, dim), generator=gen(282), device="cuda").half()
    w = torch.rand((8, heads, max(lens)), generator=gen(283), device="cuda")
    before = w.clone()
    out, lse = cache.attention(q, tables.cuda(), ints(lens), weights=w, lse=True)
    cache.check()
    for s, n in enumerate(lens):
        a = slice(s * rows, (s + 1) * rows)
        close(cache, q[a], out[a], lse[a], w[s, :, :n], before[s, :, :n], plain(cache, q[a], tables[s].tolist(), n, dim ** -0.5), n)
        assert torch.equal(w[s, :, n:], before[s, :, n:])


def test_the_largest_numbers_that_a_cache_holds(pf):
    """2^120 is the largest scale: e4m3 values of 256 and more then stand for numbers that fp32 does not have."""
    cache = pf.Kv8Cache(2, 16, 1, 64)
    x = torch.zeros((1, 1, 64), dtype=torch.bfloat16, device="cuda")
    x[0, 0, 0], x[0, 0, 1], x[0, 0, 2], x[0, 0, 3] = 3.3895313892515355e38, 3e38, -2.5e38, math.inf
    cache.append(x, x, ints([[1]]), ints([0]))
    assert (cache.scales[:, 1, 0] == 2.0 ** 120).all()
    assert cache.values[0, 1, 0, 0, :4].float().tolist() == [256.0, 224.0, -192.0, 448.0]
    cache.check()

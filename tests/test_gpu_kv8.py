"""The 8-bit KV cache on a GPU: append, attention and eviction against a plain 64-bit restatement.

Tolerances of attention, from the kernel's arithmetic (u32 = 2^-24, halves of a step of each type):
  scores   products of exact f16 operands, dim of them added in fp32 (each addition at most 2^-23 of the sum of
           magnitudes, truncation included), scaled and turned to base 2 (three roundings):
           ds = (dim + 8) * 2^-23 * spread, spread = scale * max_j sum |q k|
  p        exp2 of it: ds + 2^-21 relative; f16 for the product with V: 2^-11 more; and what is too small for that
           form by half its smallest step, 2^-22 in units of 2^-6 (up to 32 rows: four e4m3 pieces) or 2^-25 in units
           of 2^-6 (more), times V in units of the largest scale so far, at most 448 where the largest |v| is 224 or more:
           n * 2^-27 or n * 2^-30 of the largest |v|
  sums     fp32 over at most n terms: n * 2^-24
  out      sum p |v| * (2 (ds + 2^-21) + 2^-11 + 2 n 2^-24) + that + half a step of its type
"""
import math

import pytest
import torch

from tests import kv8_reference as ref

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def pf():
    if not torch.cuda.is_available():
        pytest.fail("these tests need a CUDA device (there is no CPU fallback to test)")
    import pegaflow_b200

    return pegaflow_b200


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def make_cache(pf, blocks, size, heads, dim, seed, filled=True, wide=3):
    """A cache whose every byte is set: values of every size, scales that differ by factors up to 2^wide."""
    cache = pf.Kv8Cache(blocks, size, heads, dim)
    g = gen(seed)
    if filled:
        x = torch.randn(cache.values.shape, generator=g, device="cuda") * 70
        cache.values.copy_(x.clamp(-448, 448).to(torch.float8_e4m3fn))
        cache.scales.copy_(torch.exp2(torch.randint(-7, -7 + wide + 1, cache.scales.shape, generator=g, device="cuda").float()))
    return cache


def make_tables(lens, size, seed, width=None, blocks=None):
    need = [-(-n // size) for n in lens]
    width = width or max(max(need), 1)
    total = blocks or sum(need) + 3
    ids = torch.randperm(total - 1, generator=torch.Generator().manual_seed(seed)) + 1
    t = torch.zeros((len(lens), width), dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = ids[at:at + n].int()
        at += n
    return total, t


def starts_of(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def bytes_of(cache):
    return cache.tensor.cpu().clone()


def same_bytes(cache, want, before):
    """The cache holds `want` (reference cache); every byte that is not a value or a scale is as before."""
    got = cache.values.cpu().double()
    nan = torch.isnan(want.values)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want.values[~nan])
    assert torch.equal(cache.scales.cpu().double(), want.scales)
    n = cache.kv_heads * cache.block_size * cache.head_dim + 4 * cache.kv_heads
    assert torch.equal(cache.tensor.cpu()[:, :, n:], before[:, :, n:])


# ------------------------------------------------------------------------------------------------ append
APPEND = [
    # dtype, block size, kv heads, head dim, [(old, new)]
    (torch.bfloat16, 16, 2, 128, [(0, 1), (1, 1), (15, 1), (16, 1), (17, 1), (31, 1)]),
    (torch.float16, 16, 1, 64, [(0, 16), (0, 17), (15, 2), (5, 40), (16, 15)]),
    (torch.bfloat16, 32, 3, 64, [(0, 0), (33, 0), (31, 34), (7, 1)]),
    (torch.float16, 64, 2, 256, [(63, 2), (0, 129), (70, 5)]),
    (torch.bfloat16, 128, 1, 256, [(127, 3), (0, 1), (130, 260)]),
    (torch.bfloat16, 64, 5, 128, [(200, 1)]),
    (torch.float16, 128, 2, 64, [(1, 300), (0, 0), (0, 1)]),
]


@pytest.mark.parametrize("dtype,size,heads,dim,seqs", APPEND, ids=range(len(APPEND)))
@pytest.mark.parametrize("layout", ["dense", "fused", "odd"])
def test_append(pf, dtype, size, heads, dim, seqs, layout):
    """Bit for bit: scales, new rows, old rows rounded anew; every other byte as it was."""
    lens, counts = [a for a, _ in seqs], [b for _, b in seqs]
    blocks, tables = make_tables([a + b for a, b in seqs], size, 5)
    cache = make_cache(pf, blocks, size, heads, dim, 6)
    rows = sum(counts) + 3                    # three rows behind the last sequence
    g = gen(7)
    x = torch.randn((2, rows, heads, dim), generator=g, device="cuda") * torch.exp(
        3 * torch.randn((2, rows, heads, 1), generator=g, device="cuda"))
    if layout == "dense":
        k, v = x.to(dtype).unbind(0)
    elif layout == "fused":                   # rows of K, then of V, behind query heads
        fused = torch.zeros((rows, 4 + 2 * heads, dim), dtype=dtype, device="cuda")
        fused[:, 4:4 + heads], fused[:, 4 + heads:] = x[0], x[1]
        k, v = fused[:, 4:4 + heads], fused[:, 4 + heads:]
    else:                                     # no alignment at all, heads outermost
        flat = torch.zeros((2, heads, rows, dim + 3), dtype=dtype, device="cuda")
        flat[..., 1:dim + 1] = x.transpose(1, 2)
        k, v = (flat[i].transpose(0, 1)[..., 1:dim + 1] for i in range(2))
    want, before = ref.Cache(cache), bytes_of(cache)
    starts = starts_of(counts)
    for s, (old, n) in enumerate(seqs):
        for kv, t in enumerate((k, v)):
            for h in range(heads):
                want.append(t[starts[s]:starts[s] + n, h].cpu().double(), kv, tables[s], old, h)
    cache.append(k, v, tables.cuda(), ints(lens), starts=ints(starts))
    cache.check()
    same_bytes(cache, want, before)


def test_append_special_values(pf):
    """Infinities saturate and NaN stays, neither moves the scale; zeros and the smallest numbers."""
    cache = make_cache(pf, 8, 16, 1, 64, 1)
    want, before = ref.Cache(cache), bytes_of(cache)
    x = torch.randn((6, 1, 64), generator=gen(2), device="cuda").bfloat16()
    x[0, 0, 3], x[0, 0, 4], x[0, 0, 5] = math.inf, -math.inf, math.nan
    x[1] = 0
    x[2] = 2.0 ** -130
    x[3] = 3e38
    x[4, 0, 1:] = math.inf
    x[5] = math.nan
    tables = torch.arange(1, 7, dtype=torch.int32)[:, None]
    for s in range(6):
        for kv in range(2):
            want.append(x[s:s + 1, 0].cpu().double(), kv, tables[s], 0, 0)
    cache.append(x, x, tables.cuda(), ints([0] * 6))
    cache.check()
    same_bytes(cache, want, before)


def test_append_token_by_token_gives_the_scales_of_one_call(pf):
    a, b = make_cache(pf, 9, 32, 2, 64, 3), make_cache(pf, 9, 32, 2, 64, 3)
    tables = ints([[3, 1, 7]])
    x = torch.randn((70, 2, 64), generator=gen(4), device="cuda").half() * torch.exp(torch.arange(70, device="cuda") / 20)[:, None, None].half()
    a.append(x, -x, tables, ints([0]))
    for i in range(70):
        b.append(x[i:i + 1], -x[i:i + 1], tables, ints([i]))
    assert torch.equal(a.scales[:, [3, 1, 7]], b.scales[:, [3, 1, 7]])
    # rows that were rounded twice or more: half a step each time, the scale doubling in between
    va, vb = a.values[:, 3].float() * a.scales[:, 3, :, None, None], b.values[:, 3].float() * b.scales[:, 3, :, None, None]
    assert ((va - vb).abs() <= 2.0 ** -9 * a.scales[:, 3, :, None, None]).all()


# ------------------------------------------------------------------------------------------------ attention
def check_attention(pf, cache, q, tables, lens, counts, *, causal=True, scale=None, weights=False, rows_behind=0, out=None,
                    want_cache=None, called_with=None, **kw):
    """called_with: (tables, lens) of the call where they are not those of the reference, with pages that are not there."""
    starts = starts_of(counts)
    heads, dim = cache.kv_heads, cache.head_dim
    scale_ = dim ** -0.5 if scale is None else scale
    longest = max(lens)
    w = torch.rand((len(lens), heads, longest + 5), generator=gen(99), device="cuda") if weights else None
    w0 = w.clone().cpu().double() if weights else None
    call_tables, call_lens = called_with or (tables, lens)
    got, lse = cache.attention(q, call_tables.cuda(), ints(call_lens), starts=ints(starts), max_query=max(max(counts), 1),
                               scale=scale, causal=causal, weights=w, lse=True, out=out, **kw)
    if called_with:
        with pytest.raises(pf.PegaflowInvalidArgument, match="block id"):
            cache.check()
    cache.check()
    rc = want_cache or ref.Cache(cache)
    want, want_lse, size, spread, want_w = ref.attention(q.cpu(), rc, tables, lens, starts, scale_, causal)
    n = starts[-1]
    got_, lse_ = got.cpu().double()[:n], lse.cpu().double()[:n]
    want, want_lse, size, spread = want[:n], want_lse[:n], size[:n], spread[:n]
    ds = (dim + 8) * 2.0 ** -23 * spread
    rel = 2 * (ds + 2.0 ** -21) + 2.0 ** -11 + 2 * longest * 2.0 ** -24
    big = (rc.values.abs().nan_to_num() * rc.scales[..., None, None]).max() if longest else 0.0
    tol = size * rel[..., None] + HALF[q.dtype] * want.abs() + big * longest * (2.0 ** -27 if max(counts) * q.shape[1] / heads <= 32 else 2.0 ** -30) + 1e-30
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got_), nan)
    off = ((got_ - want).abs() - tol)[~nan]
    assert off.numel() == 0 or off.max() <= 0, f"out is off by {((got_ - want).abs() / tol)[~nan].max():.3g} tolerances"
    inf = torch.isinf(want_lse)
    assert torch.equal(torch.isneginf(lse_), inf)
    lse_tol = 2 * ds + 2.0 ** -20 + 2.0 ** -22 * want_lse.abs() + longest * 2.0 ** -24
    fine = ~inf & ~torch.isnan(want_lse)
    assert (((lse_ - want_lse).abs() - lse_tol)[fine] <= 0).all()
    if weights:
        got_w = w.cpu().double()
        total = torch.zeros_like(got_w)
        for s in range(len(lens)):
            for h in range(heads):
                total[s, h, : lens[s]] = want_w[s][h]
        # both the score and lse are off by ds; rows * group terms are added, then one more to what was there
        worst = (4 * ds.max() if n else 0.0) + 2.0 ** -19 + longest * 2.0 ** -23 + max(counts) * q.shape[1] / heads * 2.0 ** -24
        assert ((got_w - (w0 + total)).abs() <= total * worst + 2.0 ** -23 * (w0 + total)).all()
    return got, lse


ATTENTION = [
    # dtype, block size, kv heads, group, head dim, lens, rows of each
    (torch.bfloat16, 16, 2, 4, 128, [1, 2, 15, 16, 17, 63, 64, 65, 300], [1] * 9),
    (torch.float16, 16, 1, 8, 64, [1000], [1]),
    (torch.bfloat16, 64, 1, 1, 64, [5, 129], [1, 1]),
    (torch.float16, 128, 3, 3, 128, [7, 200], [1, 1]),
    (torch.bfloat16, 32, 2, 5, 128, [40, 1, 300], [3, 1, 7]),
    (torch.float16, 16, 2, 7, 256, [100, 33], [1, 1]),
    (torch.bfloat16, 128, 1, 2, 256, [500], [9]),
    (torch.float16, 16, 1, 16, 128, [77, 0, 130], [1, 1, 1]),
    (torch.bfloat16, 16, 2, 1, 64, [0, 5, 0, 64], [1, 0, 3, 2]),
    (torch.bfloat16, 64, 1, 4, 128, [150], [40]),
    (torch.float16, 32, 1, 3, 64, [90, 20], [35, 20]),
    (torch.bfloat16, 16, 1, 2, 128, [3], [10]),          # more rows than tokens: the first ones see nothing
    (torch.float16, 16, 1, 4, 128, [2100], [2]),
    # around the number of rows from which on the form for many is taken
    (torch.bfloat16, 32, 1, 1, 256, [200, 17], [32, 9]),
    (torch.float16, 32, 2, 3, 64, [100, 17], [11, 9]),
    (torch.bfloat16, 16, 2, 4, 128, [300, 90], [16, 11]),
    (torch.float16, 64, 1, 2, 64, [500, 33], [24, 20]),
    (torch.bfloat16, 32, 1, 2, 256, [200, 17], [32, 9]),
    (torch.float16, 16, 1, 5, 128, [130, 0], [13, 0]),
    # many rows: tiles of 256 (128 at 256 dimensions)
    (torch.bfloat16, 16, 2, 4, 128, [700, 0, 300], [130, 0, 65]),
    (torch.float16, 64, 1, 2, 64, [1500, 128], [200, 128]),
    (torch.bfloat16, 32, 1, 1, 256, [400, 90], [150, 90]),
    (torch.bfloat16, 16, 1, 8, 128, [2000], [33]),
    (torch.float16, 128, 3, 17, 128, [257, 1], [1, 1]),
    (torch.float16, 16, 1, 3, 128, [40], [100]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,size,heads,group,dim,lens,counts", ATTENTION, ids=range(len(ATTENTION)))
def test_attention(pf, dtype, size, heads, group, dim, lens, counts, causal):
    blocks, tables = make_tables(lens, size, 11)
    cache = make_cache(pf, blocks, size, heads, dim, 12)
    q = (torch.randn((sum(counts) + 2, heads * group, dim), generator=gen(13), device="cuda") * 2).to(dtype)
    got, lse = check_attention(pf, cache, q, tables, lens, counts, causal=causal, weights=True)
    n = sum(counts)
    assert (got[n:] == 0).all() and torch.isneginf(lse[n:]).all()      # rows behind the last sequence


def test_attention_one_row_per_sequence_without_starts_and_into_a_strided_out(pf):
    lens = [30, 100, 7]
    blocks, tables = make_tables(lens, 16, 21)
    cache = make_cache(pf, blocks, 16, 2, 64, 22)
    big = torch.randn((3, 11, 64 + 4), generator=gen(23), device="cuda").bfloat16()
    q = big[:, 1:9, 1:65]                                              # no alignment
    out = torch.full((6, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    a = cache.attention(q, tables.cuda(), ints(lens))
    b = cache.attention(q, tables.cuda(), ints(lens), out=out[:3]).clone()
    c = cache.attention(q.contiguous(), tables.cuda(), ints(lens), starts=ints([0, 1, 2, 3]), max_query=1, out=out[::2])
    assert torch.equal(b, a)
    assert torch.equal(c, a)
    check_attention(pf, cache, q, tables, lens, [1, 1, 1])
    wide = torch.full((3, 8, 66), 5.0, dtype=torch.bfloat16, device="cuda")
    cache.attention(q, tables.cuda(), ints(lens), out=wide[:, :, 1:65])
    assert torch.equal(wide[:, :, 1:65], a) and (wide[:, :, 0] == 5).all() and (wide[:, :, 65] == 5).all()


def test_attention_leaves_rows_behind_the_last_sequence_of_a_given_out(pf):
    blocks, tables = make_tables([20], 16, 1)
    cache = make_cache(pf, blocks, 16, 1, 64, 2)
    q = torch.randn((8, 2, 64), generator=gen(3), device="cuda").half()
    q[1:] = math.nan
    out = torch.full_like(q, 3.0)
    cache.attention(q, tables.cuda(), ints([20]), starts=ints([0, 1]), max_query=1, out=out)
    assert (out[1:] == 3).all() and torch.isfinite(out[0]).all()


@pytest.mark.parametrize("counts", [[1], [3], [40]])
def test_attention_does_not_see_what_lies_behind_or_is_masked(pf, counts):
    """NaN in the last block behind the sequence's end, and in V and K of tokens that some rows must not see."""
    n = 75
    blocks, tables = make_tables([n], 32, 31)
    cache = make_cache(pf, blocks, 32, 1, 64, 32)
    last = int(tables[0, n // 32])
    cache.values[:, last, :, n % 32:] = torch.full((2, 1, 32 - n % 32, 64), math.nan, device="cuda").to(torch.float8_e4m3fn)
    q = torch.randn((sum(counts), 4, 64), generator=gen(33), device="cuda").half()
    got, _ = check_attention(pf, cache, q, tables, [n], counts, causal=False)
    assert torch.isfinite(got).all()
    if counts[0] > 1:      # the last token's V is NaN in one dimension: only the last row sees it
        cache.values[1, last, 0, (n - 1) % 32, 5] = torch.tensor(math.nan, device="cuda").to(torch.float8_e4m3fn)
        got, _ = check_attention(pf, cache, q, tables, [n], counts)
        assert torch.isfinite(got[:-1]).all() and torch.isnan(got[-1, :, 5]).all() and torch.isfinite(got[-1, :, :5]).all()
        cache.values[0, last, 0, (n - 1) % 32, 6] = torch.tensor(math.nan, device="cuda").to(torch.float8_e4m3fn)
        got, _ = check_attention(pf, cache, q, tables, [n], counts)
        assert torch.isfinite(got[:-1]).all() and torch.isnan(got[-1]).all()


def test_attention_over_scales_far_apart(pf):
    """Blocks whose scales differ by 2^40: the tokens that count lie in the small ones; scores of +-1000."""
    lens = [200]
    blocks, tables = make_tables(lens, 16, 41)
    cache = make_cache(pf, blocks, 16, 1, 128, 42)
    for i, b in enumerate(tables[0].tolist()):
        cache.scales[1, b] = 2.0 ** (-30 if i % 2 else 10)
        cache.scales[0, b] = 2.0 ** (-5 if i % 2 else -12)
    q = torch.randn((1, 4, 128), generator=gen(43), device="cuda").bfloat16() * 8
    check_attention(pf, cache, q, tables, lens, [1], weights=True)
    check_attention(pf, cache, (q * 2.0 ** -20), tables, lens, [1], scale=2.0 ** 18)
    check_attention(pf, cache, (q.float() * 2.0 ** 100).bfloat16(), tables, lens, [1], scale=2.0 ** -104)
    check_attention(pf, cache, q * 0, tables, lens, [1], weights=True)
    q = torch.randn((20, 4, 128), generator=gen(44), device="cuda").bfloat16() * 8
    check_attention(pf, cache, q, tables, lens, [20], weights=True)
    check_attention(pf, cache, (q * 2.0 ** -20), tables, lens, [20], scale=-2.0 ** 18)
    cache.values[1, tables[0, 4].item()] = 0               # a block of zeros: the smallest scale
    cache.scales[1, tables[0, 4].item()] = 2.0 ** -110
    check_attention(pf, cache, (q.float() * 2.0 ** 100).bfloat16(), tables, lens, [20], scale=2.0 ** -104)
    check_attention(pf, cache, q * 0, tables, lens, [20], weights=True)
    check_attention(pf, cache, q, tables, lens, [20], scale=0.0)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("order", [1, -1])
def test_attention_of_many_rows_over_scales_and_scores_that_grow(pf, dim, order):
    """Scales of K and V that rise (or fall) by 2^3 from block to block, so that nearly every step moves the unit of O, and
    scores of some rows that rise by hundreds along the sequence, so that the reference moves too."""
    lens = [400, 90]
    blocks, tables = make_tables(lens, 16, 45)
    cache = make_cache(pf, blocks, 16, 1, dim, 46)
    for s in range(2):
        for i, b in enumerate(tables[s].tolist()):
            cache.scales[1, b] = 2.0 ** (3 * order * i - 20)
            cache.scales[0, b] = 2.0 ** (order * i // 4 - 5)
    q = torch.randn((60, 2, dim), generator=gen(47), device="cuda").bfloat16()
    q[::3] *= 16
    check_attention(pf, cache, q, tables, lens, [40, 20])
    check_attention(pf, cache, q, tables, lens, [40, 20], causal=False)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("counts", [[2], [40]])
def test_attention_leaves_out_pages_that_are_not_there(pf, dim, counts):
    """Like the sequence without them, whatever block 0 and the place behind the sequence's end hold."""
    n, size = 600, 16
    blocks, tables = make_tables([n], size, 48)
    cache = make_cache(pf, blocks, size, 2, dim, 49)
    cache.values[:, 0] = torch.full((2, 2, size, dim), math.nan, device="cuda").to(torch.float8_e4m3fn)
    last = int(tables[0, n // size])
    cache.values[:, last, :, n % size:] = torch.full((2, 2, size - n % size, dim), math.nan, device="cuda").to(torch.float8_e4m3fn)
    q = torch.randn((sum(counts), 4, dim), generator=gen(50), device="cuda").half()
    called = tables.clone()
    gone = [0, 1, 2, 3, 4, 5, 6, 7, 11, 12, 30]         # the first step as a whole
    for i in gone:
        called[0, i] = -1 if i % 2 else 2 ** 30
    there = [i for i in range(-(-n // size)) if i not in gone]
    check_attention(pf, cache, q, tables[:, there].contiguous(), [n - size * len(gone)], counts, causal=False,
                    called_with=(called, [n]))


def test_weights_of_few_rows_with_and_without_room_for_their_scores(pf):
    """Tables and weights so wide that the scores of all their tokens are not kept: the same weights as in narrow ones."""
    lens, size = [70, 400], 16
    blocks, tables = make_tables(lens, size, 55)
    cache = make_cache(pf, blocks, size, 1, 128, 56)
    q = torch.randn((2, 4, 128), generator=gen(57), device="cuda").bfloat16()
    w = torch.zeros((2, 1, 400), device="cuda")
    check_attention(pf, cache, q, tables, lens, [1, 1], weights=True)
    cache.attention(q, tables.cuda(), ints(lens), weights=w)
    width = 600_000
    wide_t = torch.zeros((2, width), dtype=torch.int32, device="cuda")
    wide_t[:, :tables.shape[1]] = tables.cuda()
    wide_w = torch.zeros((2, 1, width * size), device="cuda")
    cache.attention(q, wide_t, ints(lens), weights=wide_w)
    cache.check()
    # the scores come from the same products, the exponentials from the same function of the same numbers but for their
    # rounding: 2^-20 of each, and 4 rows added
    assert torch.allclose(wide_w[:, :, :400], w, rtol=2.0 ** -19, atol=0) and (wide_w[:, :, 400:] == 0).all()


def test_weights_of_rows_whose_pages_are_not_there(pf):
    """A sequence of which nothing is there weighs nothing; the other's weights are as ever."""
    cache = make_cache(pf, 6, 16, 2, 128, 58)
    q = torch.randn((2, 4, 128), generator=gen(59), device="cuda").half()
    w = torch.zeros((2, 2, 32), device="cuda")
    cache.attention(q, ints([[77, -1], [1, 2]]), ints([30, 20]), weights=w)
    with pytest.raises(pf.PegaflowInvalidArgument, match="block id"):
        cache.check()
    assert (w[0] == 0).all() and torch.allclose(w[1].sum(-1), torch.full((2,), 2.0, device="cuda"), atol=2.0 ** -16)
    assert (w[1, :, 20:] == 0).all()


def test_attention_is_the_same_on_every_run(pf):
    lens = [700, 5000, 33]
    blocks, tables = make_tables(lens, 16, 51)
    cache = make_cache(pf, blocks, 16, 2, 128, 52)
    q = torch.randn((3, 8, 128), generator=gen(53), device="cuda").bfloat16()
    w = [torch.zeros((3, 2, 5000), device="cuda") for _ in range(2)]
    a = [cache.attention(q, tables.cuda(), ints(lens), weights=x, lse=True) for x in w]
    assert torch.equal(a[0][0], a[1][0]) and torch.equal(a[0][1], a[1][1]) and torch.equal(w[0], w[1])


def test_attention_batches_of_every_size(pf):
    """More sequences than threads of a block, empty ones among them: each like the call with it alone."""
    g = torch.Generator().manual_seed(61)
    lens = torch.randint(0, 90, (300,), generator=g).tolist()
    lens[7] = lens[200] = 0
    blocks, tables = make_tables(lens, 16, 62)
    cache = make_cache(pf, blocks, 16, 1, 64, 63)
    q = torch.randn((300, 2, 64), generator=gen(64), device="cuda").half()
    t = tables.cuda()
    got, lse = cache.attention(q, t, ints(lens), lse=True)
    check_attention(pf, cache, q, tables, lens, [1] * 300, weights=True)
    for s in (0, 7, 150, 200, 299):
        one, one_lse = cache.attention(q[s:s + 1], t[s:s + 1], ints(lens[s:s + 1]), lse=True)
        assert torch.allclose(one.float(), got[s:s + 1].float(), rtol=2.0 ** -9, atol=2.0 ** -9)
    cache.check()


# ------------------------------------------------------------------------------------------------ eviction
EVICT = [
    # block size, kv heads, head dim, lens, keep, recent
    (16, 2, 64, [1, 20, 50, 0, 100], 20, 4),
    (32, 1, 128, [300, 64], 64, 0),
    (64, 3, 256, [70, 500], 65, 65),
    (128, 2, 64, [129, 1000, 3], 130, 1),
    (16, 1, 128, [5000], 1234, 100),
    (16, 4, 64, [40, 7], 1, 0),
    (16, 1, 64, [30], 64, 10),
]


@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
@pytest.mark.parametrize("size,heads,dim,lens,keep,recent", EVICT, ids=range(len(EVICT)))
def test_evict(pf, size, heads, dim, lens, keep, recent, kind):
    blocks, tables = make_tables(lens, size, 71)
    n_dst = -(-keep // size)
    more = len(lens) * n_dst
    cache = make_cache(pf, blocks + more, size, heads, dim, 72, wide=9)
    dst = torch.arange(blocks, blocks + more, dtype=torch.int32).view(len(lens), n_dst)
    w = torch.exp(2 * torch.randn((len(lens), heads, max(lens) + 2), generator=gen(73), device="cuda"))
    if kind == "ties":
        w = torch.floor(w)
    elif kind == "special":
        w[..., ::3] = 0
        w[..., 1::7] = math.nan
        w[..., 2::11] = math.inf
        w[..., 4::13] = -0.0
        w[..., 5::17] = -1.0
    before, old = bytes_of(cache), ref.Cache(cache)
    want = ref.Cache(cache)
    new_lens, new_w, kept = cache.evict(tables.cuda(), ints(lens), w, dst.cuda(), keep, recent=recent)
    cache.check()
    assert new_lens.tolist() == [min(n, keep) for n in lens]
    w_ = w.cpu()
    for s, n in enumerate(lens):
        for h in range(heads):
            at = ref.choose(w_[s, h].tolist(), n, keep, recent)
            assert kept[s, h].tolist() == at + [-1] * (keep - len(at))
            want_w = torch.zeros(new_w.shape[2])
            want_w[: len(at)] = w_[s, h, at]
            assert torch.equal(new_w[s, h].cpu().nan_to_num(-7.0), want_w.nan_to_num(-7.0))
            for kv in range(2):
                x = old.rows(kv, tables[s], h, n)[at] if n else []
                for b in range(-(-len(at) // size)):
                    rows = {i: x[b * size + i] for i in range(min(size, len(at) - b * size))}
                    want.store(kv, int(dst[s, b]), h, rows)
    same_bytes(cache, want, before)


# ------------------------------------------------------------------------------------------------ streams, graphs, refusals
def test_other_stream_and_captured_graphs(pf):
    """Two graphs of one cache, replayed on two streams with lengths that changed in between."""
    lens = [100, 37]
    blocks, tables = make_tables([200, 200], 16, 81)
    cache = make_cache(pf, blocks, 16, 2, 128, 82)
    t, n = tables.cuda(), ints(lens)
    q = [torch.randn((2, 8, 128), generator=gen(83 + i), device="cuda").bfloat16() for i in range(2)]
    w = [torch.zeros((2, 2, 200), device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    direct = [cache.attention(x, t, n) for x in q]
    on_side = cache.attention(q[0], t, n, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(on_side, direct[0])
    graphs, outs = [], []
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(cache.attention(q[i], t, n, weights=w[i]))
        graphs.append(graph)
    for lengths in ([100, 37], [200, 1], [16, 0]):
        n.copy_(ints(lengths))
        for x in w:
            x.zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            x = torch.zeros((2, 2, 200), device="cuda")
            assert torch.equal(outs[i], cache.attention(q[i], t, n, weights=x))
            assert torch.equal(w[i], x)
    cache.check()


def test_bad_pages_lengths_and_starts_are_left_out_and_reported(pf):
    size, heads, dim = 16, 1, 64
    cache = make_cache(pf, 6, size, heads, dim, 91)
    before = bytes_of(cache)
    x = torch.randn((4, heads, dim), generator=gen(92), device="cuda").half()
    bad = ints([[1, 99], [-1, 2]])
    for call, lens, tables, starts, word in [
            ("append", [16, 0], bad, [0, 2, 4], "block id"),
            ("append", [31, -3], ints([[1, 2], [3, 4]]), [0, 2, 4], "length"),
            ("append", [1 << 30, 2147483647], ints([[1, 2], [3, 4]]), [0, 2, 4], "length"),
            ("append", [0, 0], ints([[1, 2], [3, 4]]), [0, 9, 4], "row starts"),
            ("append", [0, 0], ints([[1, 2], [3, 4]]), [-5, 1, 2147483647], "row starts"),
            ("attention", [20, 20], bad, [0, 2, 4], "block id"),
            ("attention", [33, -1], ints([[1, 2], [3, 4]]), [0, 2, 4], "length"),
            ("attention", [2147483647, 5], ints([[1, 2], [3, 4]]), [0, 2, 4], "length"),
            ("attention", [5, 5], ints([[1, 2], [3, 4]]), [0, 3, 4], "row starts"),
            ("attention", [5, 5], ints([[1, 2], [3, 4]]), [2, 1, 400], "row starts")]:
        if call == "append":
            cache.append(x, x, tables, ints(lens), starts=ints(starts))
        else:
            cache.attention(x, tables, ints(lens), starts=ints(starts), max_query=2, weights=torch.zeros((2, 1, 32), device="cuda"))
        with pytest.raises(pf.PegaflowInvalidArgument, match=word):
            cache.check()
    cache.check()                                                # reported once
    assert torch.equal(cache.tensor.cpu()[:, [0, 5]], before[:, [0, 5]])
    w = torch.rand((2, 1, 20), generator=gen(93), device="cuda")
    for lens, tables, dst, word in [([20, 20], bad, ints([[3], [4]]), "block id"), ([20, 20], ints([[1, 2], [1, 2]]), ints([[77], [4]]), "block id"),
                                    ([40, -2], ints([[1, 2], [1, 2]]), ints([[3], [4]]), "length")]:
        cache.evict(tables, ints(lens), w, dst, 8)
        with pytest.raises(pf.PegaflowInvalidArgument, match=word):
            cache.check()
    good = make_cache(pf, 6, size, heads, dim, 91)
    a = good.attention(x[:1], ints([[1, 2]]), ints([20]), weights=torch.zeros((1, 1, 10), device="cuda"))
    with pytest.raises(pf.PegaflowInvalidArgument, match="weights hold"):
        good.check()
    assert torch.equal(a, good.attention(x[:1], ints([[1, 2]]), ints([20])))


def test_refusals(pf):
    cache = pf.Kv8Cache(4, 16, 2, 64)
    t, n = ints([[1, 2]]), ints([20])
    x = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device="cuda")
    w = torch.zeros((1, 2, 32), device="cuda")
    E = pf.PegaflowInvalidArgument
    for bad, word in [
            (lambda: cache.append(x.float(), x.float(), t, n), "bfloat16 or float16"),
            (lambda: cache.append(x, x.half(), t, n), "differ"),
            (lambda: cache.append(x[:, :1], x[:, :1], t, n), "kv_heads"),
            (lambda: cache.append(x.cpu(), x, t, n), "cuda"),
            (lambda: cache.append(x, x, t.long(), n), "int32"),
            (lambda: cache.append(x, x, t, n.long()), "int32"),
            (lambda: cache.append(x, x, t, ints([1, 2])), "rows for"),
            (lambda: cache.append(x, x, t, n, starts=ints([0, 1, 1])), "2 are needed"),
            (lambda: cache.append(x.clone().requires_grad_(), x, t, n), "backward"),
            (lambda: cache.append(x, x, ints([[1], [2]]), ints([0, 0])), "evenly"),
            (lambda: cache.attention(x[:, :, ::2], t, n), "shape"),
            (lambda: cache.attention(torch.zeros((1, 2, 128), dtype=torch.half, device="cuda")[:, :, ::2], t, n), "dense"),
            (lambda: cache.attention(torch.zeros((1, 3, 64), dtype=torch.half, device="cuda"), t, n), "multiple"),
            (lambda: cache.attention(x, t, n, starts=ints([0, 1])), "max_query"),
            (lambda: cache.attention(x, t, n, max_query=0), "max_query"),
            (lambda: cache.attention(x, t, n, weights=w[:, :1]), "weights"),
            (lambda: cache.attention(x, t, n, weights=w.double()), "weights"),
            (lambda: cache.attention(x, t, n, out=x.half()), "differ"),
            (lambda: cache.evict(t, n, w, t, 8), "source"),
            (lambda: cache.evict(t, n, w, ints([[3]]), 0), "keep"),
            (lambda: cache.evict(t, n, w, ints([[3]]), 8, recent=9), "recent"),
            (lambda: cache.evict(t, n, w, ints([[3]]), 17), "does not hold"),
            (lambda: pf.Kv8Cache.from_tensor(cache.tensor[:, :, :-16], 16, 2, 64), "uint8 tensor"),
            (lambda: pf.Kv8Cache.from_tensor(cache.tensor.flatten()[1:].as_strided((2, 1, 2064), (2064, 2064, 1)), 16, 2, 64), "16 bytes"),
            (lambda: pf.Kv8Cache(4, 16, 2, 96), "head_dim"), (lambda: pf.Kv8Cache(4, 48, 2, 64), "block_size")]:
        with pytest.raises(E, match=word):
            bad()
    cache.check()
    empty = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    cache.append(empty, empty, t, n)
    assert cache.attention(empty, t, n).shape == (0, 2, 64)
    none = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    assert (cache.attention(x, none, ints([]), starts=ints([0]), max_query=1) == 0).all()
    assert cache.evict(none, ints([]), w[:0], none, 5)[0].shape == (0,)


def test_cache_in_a_slice_of_a_larger_buffer(pf):
    """Two layers in one buffer, K and V of a block next to each other: strides other than the dense ones."""
    record = pf.Kv8Cache.record_bytes(16, 2, 64)
    buffer = torch.zeros((9, 2, 2, record + 32), dtype=torch.uint8, device="cuda")      # [block, layer, K/V, record]
    layers = [pf.Kv8Cache.from_tensor(buffer[:, i].transpose(0, 1), 16, 2, 64) for i in range(2)]
    dense = [pf.Kv8Cache(9, 16, 2, 64) for _ in range(2)]
    t, n = ints([[4, 2, 8]]), ints([0])
    for i in range(2):
        x = torch.randn((2, 40, 2, 64), generator=gen(i), device="cuda").half()
        for c in (layers[i], dense[i]):
            c.append(x[0], x[1], t, n)
    q = torch.randn((1, 4, 64), generator=gen(5), device="cuda").half()
    for a, b in zip(layers, dense):
        assert torch.equal(a.values.float(), b.values.float()) and torch.equal(a.scales, b.scales)
        assert torch.equal(a.attention(q, t, ints([40])), b.attention(q, t, ints([40])))
    assert (buffer[..., record:] == 0).all()


# ------------------------------------------------------------------------------------------------ together
def test_prompt_decode_evict_offload_and_reload(pf):
    """A prompt is written, decoded with its weights kept, cut to a budget, saved to the pool, loaded into other blocks of
    another cache and decoded on: every step against the restatement, the reloaded cache bit for bit."""
    from pegaflow_b200 import connector

    size, heads, group, dim, blocks = 16, 2, 4, 128, 64
    names = ["l0", "l1"]
    src = {n: pf.Kv8Cache(blocks, size, heads, dim) for n in names}
    dst = {n: pf.Kv8Cache(blocks, size, heads, dim) for n in names}
    g = gen(101)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:12].int()[None] + 1
    short = torch.arange(45, 49, dtype=torch.int32)[None]
    prompt, keep = 150, 60
    for name in names:
        c = src[name]
        kv = torch.randn((2, prompt, heads, dim), generator=g, device="cuda").bfloat16()
        c.append(kv[0], kv[1], table.cuda(), ints([0]))
        w = torch.zeros((1, heads, size * 12), device="cuda")
        n = prompt
        for _ in range(5):
            kv = torch.randn((2, 1, heads, dim), generator=g, device="cuda").bfloat16()
            c.append(kv[0], kv[1], table.cuda(), ints([n]))
            n += 1
            q = torch.randn((1, heads * group, dim), generator=g, device="cuda").bfloat16()
            c.attention(q, table.cuda(), ints([n]), weights=w)
            check_attention(pf, c, q, table, [n], [1])
        assert torch.allclose(w.sum(-1), torch.full((1, heads), 5.0 * group, device="cuda"), rtol=1e-4)
        lens, w, kept = c.evict(table.cuda(), ints([n]), w, short.cuda(), keep, recent=8)
        assert lens.tolist() == [keep] and (w[..., keep:] == 0).all() and kept[0, 0, -1] == n - 1
        c.check()
    eng = pf.PegaEngine(64 << 20)
    client = connector.InProcEngineClient(eng)
    hashes = [b"kv8-%d" % i for i in range(4)]
    conns = []
    for who, caches in (("a", src), ("b", dst)):
        conn = connector.PegaWorkerConnector(client, eng, instance_id=who, namespace="kv8", device_id=0, block_size=size)
        conn.register_kv_caches(caches)
        conns.append(conn)
    torch.cuda.synchronize()
    conns[0].wait_for_save([(n, short[0].tolist(), hashes) for n in names])
    hit = client.query_prefetch("b", hashes, "r")
    assert hit.num_hit_blocks == 4
    home = [9, 3, 30, 11]
    conns[1].start_load_kv([("r", hit.lease, home)])
    done = []
    while not done:
        done, failed = conns[1].get_finished()
        assert not failed
    for name in names:
        a, b = src[name], dst[name]
        assert torch.equal(a.tensor[:, short[0].long().cuda()], b.tensor[:, home])
        t = torch.tensor([home], dtype=torch.int32)
        kv = torch.randn((2, 3, heads, dim), generator=g, device="cuda").bfloat16()
        b.append(kv[0], kv[1], t.cuda(), ints([keep]))
        q = torch.randn((3, heads * group, dim), generator=g, device="cuda").bfloat16()
        check_attention(pf, b, q, t, [keep + 3], [3], weights=True)
    for conn in conns:
        conn.unregister()
    eng.close()

"""The 8-bit KV cache's operators as a benchmark: listed and drawn cases of the write (append), the attention that
reads the cache, and the eviction by accumulated attention weight.  ``own`` chooses between the plain form in
elementary torch operations and the framework's own kernels."""
import math

import torch

own = False

E4M3_MAX = 448.0
E_MIN, E_MAX = -110, 120


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One decode step's write of a serving batch: one token for each of 32 requests, the smallest call there is.
        {"name": "append-decode-32", "op": "append", "batch": 32, "old_lo": 1, "old_hi": 4000, "new_lo": 1, "new_hi": 1,
         "kv_heads": 8, "head_dim": 128, "block": 16, "dtype": "bfloat16"},
        # The write of a mixed step of a small model: odd chunks behind odd prefixes, blocks of 64, half precision.
        {"name": "append-ragged-13", "op": "append", "batch": 13, "old_lo": 0, "old_hi": 1999, "new_lo": 1, "new_hi": 1777,
         "kv_heads": 2, "head_dim": 64, "block": 64, "dtype": "float16"},
        # A cold prefill of the benchmark's prompts: 8 requests of 10240 tokens into empty blocks.
        {"name": "append-prefill-8x10240", "op": "append", "batch": 8, "old_lo": 0, "old_hi": 0, "new_lo": 10240, "new_hi": 10240,
         "kv_heads": 8, "head_dim": 128, "block": 16, "dtype": "bfloat16"},
        # One request's decode step over a short context: launch and join latency.
        {"name": "decode-1x1000", "op": "attention", "batch": 1, "len_lo": 1000, "len_hi": 1000, "new_lo": 1, "new_hi": 1,
         "kv_heads": 8, "group": 4, "head_dim": 128, "block": 16, "dtype": "bfloat16", "weights": False},
        # Decode step of the benchmark's batch, 8 prompts of 10240 tokens, keeping the weights that eviction goes by.
        {"name": "decode-8x10240-weights", "op": "attention", "batch": 8, "len_lo": 10240, "len_hi": 10240, "new_lo": 1,
         "new_hi": 1, "kv_heads": 8, "group": 4, "head_dim": 128, "block": 16, "dtype": "bfloat16", "weights": True},
        # Decode step of a full serving batch whose contexts differ by more than a factor of ten.
        {"name": "decode-48-ragged", "op": "attention", "batch": 48, "len_lo": 700, "len_hi": 16001, "new_lo": 1, "new_hi": 1,
         "kv_heads": 8, "group": 4, "head_dim": 128, "block": 16, "dtype": "bfloat16", "weights": False},
        # One very long context on one rank of a tensor-parallel model: a single KV head pair, heads of 64, blocks of 64.
        {"name": "decode-1x131000", "op": "attention", "batch": 1, "len_lo": 131000, "len_hi": 131000, "new_lo": 1, "new_hi": 1,
         "kv_heads": 2, "group": 8, "head_dim": 64, "block": 64, "dtype": "float16", "weights": False},
        # Verification of drafted tokens: a few queries for each request, the group of 5 does not fill a tile.
        {"name": "verify-16-ragged", "op": "attention", "batch": 16, "len_lo": 300, "len_hi": 9000, "new_lo": 2, "new_hi": 7,
         "kv_heads": 4, "group": 5, "head_dim": 128, "block": 32, "dtype": "bfloat16", "weights": False},
        # A warm request: the prompt's first 10240 tokens were loaded, the 2048 behind them are computed now.
        {"name": "suffix-2048-on-10240", "op": "attention", "batch": 1, "len_lo": 12288, "len_hi": 12288, "new_lo": 2048,
         "new_hi": 2048, "kv_heads": 8, "group": 4, "head_dim": 128, "block": 16, "dtype": "bfloat16", "weights": False},
        # One request over its budget: the smallest eviction.
        {"name": "evict-1x1500-to-512", "op": "evict", "batch": 1, "len_lo": 1500, "len_hi": 1500, "keep": 512, "recent": 64,
         "kv_heads": 8, "head_dim": 128, "block": 16},
        # A batch of unequal requests, some within the budget already.
        {"name": "evict-11-ragged-to-777", "op": "evict", "batch": 11, "len_lo": 200, "len_hi": 7001, "keep": 777, "recent": 100,
         "kv_heads": 4, "head_dim": 64, "block": 64},
        # The benchmark's prompts cut to two fifths before they are offloaded.
        {"name": "evict-16x10240-to-4096", "op": "evict", "batch": 16, "len_lo": 10240, "len_hi": 10240, "keep": 4096,
         "recent": 512, "kv_heads": 8, "head_dim": 128, "block": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "evict"])
    c = {"op": op, "kv_heads": rng.choice([1, 2, 3, 4, 8]), "head_dim": rng.choice([64, 128, 128, 256]),
         "block": rng.choice([16, 16, 32, 64, 128]), "dtype": rng.choice(["bfloat16", "float16"])}
    row = c["kv_heads"] * c["head_dim"]
    if op == "append":
        c["batch"] = _log(rng, 1, 64)
        top = max(1, min(10240, 80_000_000 // (row * c["batch"])))
        c["new_hi"] = _log(rng, 1, top)
        c["new_lo"] = rng.randint(1, c["new_hi"])
        c["old_lo"], c["old_hi"] = 0, _log(rng, 1, 8000)
    elif op == "attention":
        c["group"] = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        c["weights"] = rng.random() < 0.3
        form = rng.choice(["decode", "decode", "verify", "suffix"])
        c["batch"] = _log(rng, 1, 64) if form != "suffix" else _log(rng, 1, 8)
        c["len_hi"] = _log(rng, 1, max(1, min(131072, 240_000_000 // (row * c["batch"]))))
        c["len_lo"] = rng.randint(max(1, c["len_hi"] // 20), c["len_hi"])
        c["new_hi"] = 1 if form == "decode" else rng.randint(2, 16) if form == "verify" else _log(rng, 17, 2048)
        heads = c["kv_heads"] * c["group"]
        pairs = min(800_000_000, 90_000_000_000 // c["head_dim"])           # the plain form holds a score for each
        most = pairs // (c["batch"] * heads * c["len_hi"])
        c["new_hi"] = max(1, min(c["new_hi"], most, c["len_hi"]))
        c["new_lo"] = rng.randint(max(1, c["new_hi"] // 2), c["new_hi"])
    else:
        del c["dtype"]
        c["batch"] = _log(rng, 1, 32)
        c["len_hi"] = _log(rng, 2, max(2, min(65536, 80_000_000 // (row * c["batch"]))))
        c["len_lo"] = rng.randint(1, c["len_hi"])
        c["keep"] = max(1, int(c["len_hi"] * rng.uniform(0.1, 0.8)))
        c["recent"] = rng.randint(0, c["keep"])
    return c


def _spread(lo, hi, n, turn):
    """n lengths between lo and hi, the same for every seed: spread evenly over the logarithm, in mixed order."""
    if n == 1:
        return [hi]
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [int(round(math.exp(a + (b - a) * ((i * turn) % n) / (n - 1)))) - 1 for i in range(n)]


def _turn(n):
    return next(t for t in (7, 11, 13, 17, 19, 23) if math.gcd(t, n) == 1)


def _lengths(case):
    """(new tokens, length behind which they stand or that they are part of) for each sequence."""
    n = case["batch"]
    if case["op"] == "evict":
        return None, _spread(case["len_lo"], case["len_hi"], n, _turn(n))
    new = _spread(case["new_lo"], case["new_hi"], n, 1)
    if case["op"] == "append":
        return new, _spread(case["old_lo"], case["old_hi"], n, _turn(n))
    return new, [max(a, b) for a, b in zip(new, _spread(case["len_lo"], case["len_hi"], n, _turn(n)))]


def _record(case):
    """(bytes of the values, bytes of a whole record) of one block of K or V."""
    values = case["kv_heads"] * case["block"] * case["head_dim"]
    return values, values + (4 * case["kv_heads"] + 15) // 16 * 16


def work(case):
    new, lens = _lengths(case)
    heads, dim = case["kv_heads"], case["head_dim"]
    blocks = sum(-(-n // case["block"]) for n in lens)
    if case["op"] == "append":
        n = sum(new)
        return {"bytes": n * heads * dim * 2 * 3, "flops": n * heads * dim * 2 * 2}
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        candidates = sum(lens) * heads
        return {"bytes": 4 * candidates + heads * kept * (4 * dim + 8), "flops": candidates + heads * kept * dim * 4}
    pairs = sum(n * q - q * (q - 1) // 2 for q, n in zip(new, lens))
    q_bytes = sum(new) * heads * case["group"] * dim * 2 * 2
    kv = sum(lens) * heads * dim * 2 + blocks * heads * 8
    return {"bytes": kv + q_bytes + (8 * sum(lens) * heads if case["weights"] else 0),
            "flops": 4 * dim * heads * case["group"] * pairs}


# ---------------------------------------------------------------------------------------------- inputs
def _cache(case, blocks, gen, filled):
    """uint8 [2, blocks, record]: e4m3 values [kv_heads, block, head_dim], then one power-of-two scale for each head."""
    heads, size, dim = case["kv_heads"], case["block"], case["head_dim"]
    values, record = _record(case)
    t = torch.zeros((2, blocks, record), dtype=torch.uint8, device="cuda")
    if filled:
        x = torch.randn((2, blocks, values), generator=gen, device="cuda", dtype=torch.bfloat16) * 60
        t[:, :, :values] = x.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
        e = torch.randint(-7, -4, (2, blocks, heads), generator=gen, device="cuda")
        _scales(t, case).copy_(torch.exp2(e.float()))
    return t


def _values(t, case):
    values, _ = _record(case)
    return t[:, :, :values].view(2, t.shape[1], case["kv_heads"], case["block"], case["head_dim"])


def _scales(t, case):
    values, _ = _record(case)
    return t[:, :, values:values + 4 * case["kv_heads"]].view(torch.float32)


def _tables(case, lens, gen, spare=0):
    """Block tables of randomly placed blocks (int32 [batch, most]) for `lens` tokens, and for `spare` more for each."""
    size, n = case["block"], len(lens)
    need = [-(-v // size) for v in lens]
    most, most_spare = max(max(need), 1), -(-spare // size)
    total = n * (most + most_spare) + 1
    ids = torch.randperm(total - 1, generator=gen, device="cuda").to(torch.int32) + 1
    src = ids[: n * most].view(n, most).clone()
    past = torch.arange(most, device="cuda") >= torch.tensor(need, device="cuda")[:, None]
    src[past] = 0
    return total, src, ids[n * most:].view(n, most_spare).clone() if spare else None


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    new, lens = _lengths(case)
    heads, dim = case["kv_heads"], case["head_dim"]
    s = {"case": case, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    if case["op"] == "evict":
        blocks, s["tables"], s["dst"] = _tables(case, lens, gen, case["keep"])
        s["cache"] = _cache(case, blocks, gen, True)
        w = torch.exp(torch.randn((case["batch"], heads, max(lens)), generator=gen, device="cuda") * 2)
        # tokens that attention never looked at have no weight at all: they tie
        s["weights"] = w * (torch.rand(w.shape, generator=gen, device="cuda") > 0.3)
        return s
    dtype = getattr(torch, case["dtype"])
    total = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["max_new"] = max(new)
    if case["op"] == "append":
        blocks, s["tables"], _ = _tables(case, [a + b for a, b in zip(new, lens)], gen)
        s["cache"] = _cache(case, blocks, gen, True)
        kv = torch.randn((total, 2, heads, dim), generator=gen, device="cuda") * 1.5
        kv *= torch.exp(torch.randn((1, 2, heads, dim), generator=gen, device="cuda") * 0.5)      # channels differ in size
        s["k"], s["v"] = kv.to(dtype).unbind(1)          # as a fused projection leaves them: rows of K, then of V
        return s
    blocks, s["tables"], _ = _tables(case, lens, gen)
    s["cache"] = _cache(case, blocks, gen, True)
    s["q"] = (torch.randn((total, heads * case["group"], dim), generator=gen, device="cuda") * 1.5).to(dtype)
    s["scale"] = dim ** -0.5
    if case["weights"]:
        s["weights"] = torch.rand((case["batch"], heads, max(lens)), generator=gen, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------- one pass
def _handle(s):
    """The cache object that a program keeps for its layer."""
    if "handle" not in s:
        import pegaflow_b200 as pf

        c = s["case"]
        s["handle"] = pf.Kv8Cache.from_tensor(s["cache"], c["block"], c["kv_heads"], c["head_dim"])
    return s["handle"]


def run(s):
    case = s["case"]
    if own:
        cache = _handle(s)
        if case["op"] == "append":
            cache.append(s["k"], s["v"], s["tables"], s["lens"], starts=s["starts"])
            return {"values": cache.values, "scales": cache.scales}
        if case["op"] == "evict":
            lens, weights, kept = cache.evict(s["tables"], s["lens"], s["weights"], s["dst"], case["keep"], recent=case["recent"])
            return {"lens": lens, "weights": weights, "kept": kept, "values": cache.values, "scales": cache.scales}
        weights = s["weights"].clone() if case["weights"] else None
        out, lse = cache.attention(s["q"], s["tables"], s["lens"], starts=s["starts"], max_query=s["max_new"], scale=s["scale"],
                                   weights=weights, lse=True)
        return {"out": out, "lse": lse, "weights": weights}
    return {"append": _plain_append, "attention": _plain_attention, "evict": _plain_evict}[case["op"]](s)


def _exponent(amax):
    """Least e with amax <= 448 * 2^e, clamped; amax in 32 bits."""
    m, x = torch.frexp(amax)                     # amax = m * 2^x, m in [0.5, 1); 448 = 0.875 * 2^9
    e = x - 9 + (m > 0.875).to(x.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _f8(u8):
    return u8.view(torch.float8_e4m3fn).float()


def _outputs(s):
    case = s["case"]
    return {"values": _values(s["cache"], case).view(torch.float8_e4m3fn), "scales": _scales(s["cache"], case)}


def _plain_append(s):
    case, starts, size = s["case"], s["starts"].long(), s["case"]["block"]
    total = s["k"].shape[0]
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    pos = s["lens"].long()[seq] + row - starts[seq]
    block, off = s["tables"].long()[seq, pos // size], pos % size
    x = torch.stack([s["k"], s["v"]]).float()                                   # [2, total, heads, dim]
    values, scales = _values(s["cache"], case), _scales(s["cache"], case)
    index = block[None, :, None].expand(2, total, case["kv_heads"])
    e_new = torch.full(scales.shape, E_MIN, dtype=torch.int32, device="cuda").scatter_reduce(
        1, index, _exponent(x.abs().amax(-1)), "amax")
    # rows of the first block that were there before
    has = torch.zeros(scales.shape[1], dtype=torch.int64, device="cuda")
    first = s["lens"].long() % size
    live = (first > 0) & (starts[1:] > starts[:-1])
    at = s["tables"].long().gather(1, (s["lens"].long() // size).clamp(max=s["tables"].shape[1] - 1)[:, None])[:, 0]
    has.scatter_reduce_(0, at, torch.where(live, first, torch.zeros_like(first)), "amax")
    touched = torch.zeros(scales.shape[1], dtype=torch.bool, device="cuda").index_fill(0, block, True)
    e_old = torch.frexp(scales)[1] - 1
    e = torch.where((has > 0)[None, :, None], torch.maximum(e_old, e_new), e_new)
    part = torch.nonzero(has > 0)[:, 0]
    old = _f8(values[:, part]) * torch.exp2((e_old - e)[:, part].float())[..., None, None]
    keep = (torch.arange(size, device="cuda") < has[part][:, None])[None, :, None, :, None]
    values[:, part] = torch.where(keep, old.to(torch.float8_e4m3fn).view(torch.uint8), values[:, part])
    scales.copy_(torch.where(touched[None, :, None], torch.exp2(e.float()), scales))
    y = x * torch.exp2(-e.float())[:, block][..., None]
    values[:, block, :, off] = y.to(torch.float8_e4m3fn).view(torch.uint8).transpose(0, 1)
    return _outputs(s)


def _rows(s, kv, pos):
    """Values in 32 bits at positions `pos` ([batch, ..., n], heads in between if any): [batch, heads, n, dim]."""
    case, size = s["case"], s["case"]["block"]
    values, scales = _values(s["cache"], case)[kv], _scales(s["cache"], case)[kv]
    head = torch.arange(case["kv_heads"], device="cuda")[None, :, None]
    seq = torch.arange(pos.shape[0], device="cuda")[:, None, None]
    block = s["tables"].long()[seq, pos // size]
    return _f8(values[block, head, pos % size]) * scales[block, head][..., None]


def _plain_attention(s):
    case = s["case"]
    batch, heads, group = case["batch"], case["kv_heads"], case["group"]
    lens, starts, most = s["lens"].long(), s["starts"].long(), s["max_new"]
    new = starts[1:] - starts[:-1]
    j = torch.arange(int(s["tables"].shape[1]) * case["block"], device="cuda")[: case["len_hi"] if case["len_hi"] > most else most]
    pos = j[None, None].expand(batch, heads, -1)
    i = torch.arange(most, device="cuda")
    rows = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(batch, most, heads, group, -1).permute(0, 2, 1, 3, 4).reshape(batch, heads, most * group, -1)
    see = (j[None, None] <= (lens - new)[:, None, None] + i[None, :, None]) & (j[None, None] < lens[:, None, None])   # [batch, most, n]
    see = see[:, None, :, None].expand(batch, 1, most, group, -1).reshape(batch, 1, most * group, -1)
    x = torch.matmul(q, _rows(s, 0, pos).transpose(-1, -2)).mul_(s["scale"])
    x.masked_fill_(~see, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    lse = torch.log(total) + top
    x /= total.clamp(min=1e-30)
    live = (i[None] < new[:, None])
    back = lambda t: t.view(batch, heads, most, group, -1).permute(0, 2, 1, 3, 4)[live].reshape(s["q"].shape[0], heads * group, -1)  # noqa: E731
    weights = None
    if case["weights"]:
        x2 = x * live[:, None, :, None].expand(batch, 1, most, group).reshape(batch, 1, most * group, 1)
        weights = s["weights"] + x2.sum(2)
    out = torch.matmul(x, _rows(s, 1, pos))
    return {"out": back(out).to(s["q"].dtype), "lse": back(lse)[..., 0], "weights": weights}


def _plain_evict(s):
    case, size, keep = s["case"], s["case"]["block"], s["case"]["keep"]
    lens, w = s["lens"].long()[:, None, None], s["weights"]
    batch, heads, most = w.shape
    j = torch.arange(most, device="cuda")
    kept_n = lens.clamp(max=keep)
    recent = lens.clamp(max=case["recent"])
    candidate = j < lens - recent
    order = torch.sort(torch.where(candidate, w, torch.full_like(w, -1)), dim=-1, descending=True, stable=True)[1]
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order))
    chosen = (candidate & (rank < kept_n - recent)) | ((j >= lens - recent) & (j < lens))
    kept = torch.sort(torch.where(chosen, j, torch.full_like(order, most)), dim=-1)[0]
    kept = torch.nn.functional.pad(kept, (0, max(0, keep - most)), value=most)[..., :keep]
    valid = kept < most
    pos = torch.where(valid, kept, torch.zeros_like(kept))
    weights = torch.zeros_like(w)
    weights[..., :keep] = torch.where(valid, w.gather(-1, pos), torch.zeros_like(pos, dtype=w.dtype))[..., :most]
    n_dst = -(-keep // size)
    pad = n_dst * size - keep
    full = torch.nn.functional.pad(valid, (0, pad)).view(batch, heads, n_dst, size)
    dst = s["dst"].long()
    values, scales = _values(s["cache"], case), _scales(s["cache"], case)
    x = torch.stack([_rows(s, 0, pos), _rows(s, 1, pos)])
    x = torch.nn.functional.pad(x, (0, 0, 0, pad)).view(2, batch, heads, n_dst, size, -1)
    x = x * full[None, ..., None]
    e = _exponent(x.abs().amax((-1, -2)))                                                # [2, batch, heads, n_dst]
    y = (x * torch.exp2(-e.float())[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    y = y.permute(0, 1, 3, 2, 4, 5)                                                      # [2, batch, n_dst, heads, size, dim]
    mask = full.permute(0, 2, 1, 3)[None, ..., None]
    values[:, dst] = torch.where(mask, y, values[:, dst])
    used = full.any(-1).permute(0, 2, 1)[None]
    scales[:, dst] = torch.where(used, torch.exp2(e.permute(0, 1, 3, 2).float()), scales[:, dst])
    return {"lens": kept_n[:, 0, 0].int(), "weights": weights, "kept": torch.where(valid, kept, torch.full_like(kept, -1)).int(),
            **_outputs(s)}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "evict": _exact_evict}[case["op"]](s)


def _real(s, kv, seq, head, n):
    """The first n rows that sequence `seq` holds for one head, as the numbers they stand for, in 64 bits."""
    case, size = s["case"], s["case"]["block"]
    ids = s["tables"][seq, : -(-n // size)].long()
    t = s["cache"][kv, ids]
    one = size * case["head_dim"]
    values = t[:, head * one:(head + 1) * one].contiguous().view(torch.float8_e4m3fn).double().view(-1, size, case["head_dim"])
    at = case["kv_heads"] * one + 4 * head
    scale = t[:, at:at + 4].contiguous().view(torch.float32).double()
    return (values * scale[:, :, None]).reshape(-1, case["head_dim"])[:n]


def _scale64(top):
    """The scale that a largest magnitude asks for."""
    if not top > 0:
        return 2.0 ** E_MIN
    e = math.ceil(math.log2(top / E4M3_MAX))
    e -= top <= E4M3_MAX * 2.0 ** (e - 1)
    e += top > E4M3_MAX * 2.0 ** e
    return 2.0 ** min(max(e, E_MIN), E_MAX)


def _exact_append(s):
    case, size, dim = s["case"], s["case"]["block"], s["case"]["head_dim"]
    if s["k"].shape[0] * case["kv_heads"] > 60000:                   # block by block it would take too long
        return None
    values = _values(s["cache"], case).view(torch.float8_e4m3fn).double()
    scales = _scales(s["cache"], case).double()
    starts, lens, tables = s["starts"].tolist(), s["lens"].tolist(), s["tables"].tolist()
    for kv, x in enumerate((s["k"], s["v"])):
        tops = x.double().abs().amax(-1).cpu()
        for seq, old in enumerate(lens):
            p, at = old, starts[seq]
            while at < starts[seq + 1]:
                block, row = tables[seq][p // size], p % size
                n = min(size - row, starts[seq + 1] - at)
                want = torch.tensor([_scale64(v) for v in tops[at:at + n].amax(0).tolist()], dtype=torch.float64, device="cuda")
                if row:
                    was = scales[kv, block].clone()
                    want = torch.maximum(want, was)
                    values[kv, block, :, :row] *= (was / want)[:, None, None]
                scales[kv, block] = want
                values[kv, block, :, row:row + n] = x[at:at + n].double().transpose(0, 1) / want[:, None, None]
                p, at = p + n, at + n
    return {"values": values, "scales": scales}


def _exact_attention(s):
    case, group = s["case"], s["case"]["group"]
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if case["weights"] else None
    for seq, n in enumerate(lens):
        a, b = starts[seq], starts[seq + 1]
        last = n - (b - a) + torch.arange(b - a, device="cuda")
        hidden = torch.arange(n, device="cuda")[None] > last[:, None]
        for head in range(case["kv_heads"]):
            k, v = _real(s, 0, seq, head, n), _real(s, 1, seq, head, n)
            for g in range(head * group, (head + 1) * group):
                x = (s["q"][a:b, g].double() @ k.T * s["scale"]).masked_fill(hidden, -math.inf)
                lse[a:b, g] = torch.logsumexp(x, -1)
                p = torch.softmax(x, -1)
                out[a:b, g] = p @ v
                if weights is not None:
                    weights[seq, head, :n] += p.sum(0)
    return {"out": out, "lse": lse, "weights": weights}


def _exact_evict(s):
    case, size, keep = s["case"], s["case"]["block"], s["case"]["keep"]
    values = _values(s["cache"], case).view(torch.float8_e4m3fn).double()
    scales = _scales(s["cache"], case).double()
    weights = torch.zeros_like(s["weights"], dtype=torch.float64)
    lens, w, dst = s["lens"].tolist(), s["weights"].double().cpu(), s["dst"].tolist()
    for seq, n in enumerate(lens):
        recent = min(case["recent"], n)
        for head in range(case["kv_heads"]):
            old = w[seq, head, : n - recent]
            best = torch.argsort(old, descending=True, stable=True)[: max(0, min(keep, n) - recent)]
            at = torch.cat([best.sort()[0], torch.arange(n - recent, n)])
            weights[seq, head, : at.numel()] = s["weights"][seq, head, at.cuda()].double()
            for kv in range(2):
                x = _real(s, kv, seq, head, n)[at.cuda()]
                m = -(-x.shape[0] // size)
                if not m:
                    continue
                ids = torch.tensor(dst[seq][:m], device="cuda")
                x = torch.nn.functional.pad(x, (0, 0, 0, m * size - x.shape[0])).view(m, size, -1)
                new = torch.tensor([_scale64(t) for t in x.abs().amax((1, 2)).tolist()], dtype=torch.float64, device="cuda")
                scales[kv, ids, head] = new
                whole = values[kv, ids, head]
                flat = whole.view(m * size, -1)
                flat[: at.numel()] = (x / new[:, None, None]).view(m * size, -1)[: at.numel()]
                values[kv, ids, head] = whole
    return {"lens": None, "weights": weights, "kept": None, "values": values, "scales": scales}

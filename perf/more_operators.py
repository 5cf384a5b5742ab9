"""Rotary appends and the 8-bit KV cache's operators as measurable cases: new
keys and values rotated by their positions on their way into the 16-bit cache
and into the 8-bit one, the 8-bit cache's de-page, its decode attention and its
attention of several query tokens per sequence, all over blocks of 16 tokens.

``listed`` names the cases, ``draw`` makes more of the same ranges, ``prepare``
makes what a program has in hand before the call, ``run`` is one pass (the
operators' plain form, or with ``own`` the framework's calls), ``work`` the
bytes and operations a pass cannot do without, ``exact`` the outputs in 64 bits.

The rotation.  ``table [positions, R]`` float32 holds the cosines of a
position's R/2 angles, then their sines.  Of the first R dims of a row, dims i
and i + R/2 (``inter``: 2 i and 2 i + 1) are a pair (x, y) and become
(x cos - y sin, y cos + x sin) of angle i; the dims past R stay.

The 8-bit cache's numbers.  The 16 tokens of a block share, per head and side
(K or V), an exponent e: the least integer with max|x| <= 448 * 2^e over the
block's finite values, within [-117, 119] (bf16) or [-15, 7] (fp16).  A value's
code is x / 2^e rounded to the nearest number of four exponent and three
mantissa bits (ties to even, at most 448; NaN for an infinity or a NaN).  Tokens
that join a block which has earlier ones take the larger of its exponent and
their own; if it rises, the earlier tokens' values are rounded once more to its
codes.  A token at a block's first place begins the block anew.

The 8-bit cache's bytes.  ``[N, L, 32 Hkv D + 4 Hkv, padded to 128]`` uint8: per
head K's 16 D codes and V's, then 4 bytes per head (K's e + 127, V's, two more).
K codes ``[chunk of 16 dims][16 tokens][16 dims]``; V codes ``[D/64 pieces][4
token quads][16 lanes][4 dims][4 tokens]``, lane j holding dims D/16 j .. of
which piece i has 4 i .. 4 i + 3.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 16  # tokens per block
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOP = {torch.bfloat16: 119, torch.float16: 7}     # largest exponent of a block
LOW = {torch.bfloat16: -117, torch.float16: -15}  # and least
LARGEST = 448.0                                   # of a code
BASE = 10000.0                                    # of the angles' geometric series


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _case(name, kind, dtype, hq, hkv, dim, layers, seqs, mean, sigma, lo, hi, lens_seed=0, **more):
    """``seqs`` sequences whose lengths are lognormal with arithmetic mean
    ``mean`` and ``sigma``, clipped to [lo, hi]; sigma 0: all ``mean``."""
    return dict(name=name, kind=kind, dtype=dtype, hq=hq, hkv=hkv, dim=dim, layers=layers,
                seqs=seqs, mean=mean, sigma=sigma, lo=lo, hi=hi, lens_seed=lens_seed, **more)


def listed():
    return [
        # One layer of a decode step: the queries and new keys of 128 sequences
        # rotated, keys and values written to the 16-bit cache.
        _case("rotary_step_qwen_128", "rotary", "bf16", 28, 4, 128, 1, 128, 200, 0.5, 1, 1000,
              whole=False, rot=128, inter=False),
        # One layer of a prompt run, the rotated keys kept for the prompt's own
        # attention too; pairs of neighbours, half of the dims rotated.
        _case("rotary_prompt_4x1000", "rotary", "fp16", 32, 4, 128, 1, 4, 1000, 0.1, 1, 1100,
              whole=True, rot=64, inter=True),
        # One layer of a decode step into the 8-bit cache, whose open blocks
        # are then read back, as an engine does that hands them on in 16 bits.
        _case("append8_step_qwen_128", "append8", "bf16", 28, 4, 128, 1, 128, 40, 0.5, 1, 96,
              whole=False, rot=128, inter=False),
        # One layer of four prompts of uneven lengths, and what it stands for.
        _case("append8_prompt_4x1000", "append8", "bf16", 28, 4, 128, 1, 4, 1000, 0.1, 1, 1100,
              whole=True, rot=128, inter=False),
        # De-page of a batch of very different lengths, one layer.
        _case("gather8_qwen_128", "gather8", "bf16", 28, 4, 128, 1, 128, 400, 1.0, 16, 4096),
        # The same for a few short sequences of wide heads: latency.
        _case("gather8_wide_6", "gather8", "fp16", 6, 2, 256, 1, 6, 50, 0.8, 1, 128),
        # The smallest decode attention: one layer, eight short sequences.
        _case("decode8_tiny", "decode8", "fp16", 2, 2, 64, 1, 8, 60, 0.8, 1, 128),
        # A loaded engine: 128 sequences of very different lengths, one plan
        # for four layers of the step.
        _case("decode8_qwen_128", "decode8", "bf16", 28, 4, 128, 4, 128, 1500, 1.0, 16, 8192),
        # Multi-head attention without grouping: the most cached bytes per token.
        _case("decode8_llama_32", "decode8", "fp16", 40, 40, 128, 1, 32, 1999, 0.0, 1, 4096),
        # One very long context: one sequence over the whole chip.
        _case("decode8_long_context", "decode8", "bf16", 28, 4, 128, 2, 1, 131001, 0.0, 1, 131072),
        # Five drafted tokens per sequence checked at once.
        _case("varlen8_draft_48", "varlen8", "fp16", 32, 4, 128, 1, 48, 1000, 0.8, 16, 4096,
              new=5, causal=True),
        # The last chunk of one long document.
        _case("varlen8_document", "varlen8", "bf16", 28, 4, 128, 1, 1, 16001, 0.0, 1, 16384,
              new=2048, causal=True),
    ]


# (query heads, kv heads, head dim) of the framework's models and tests
_SHAPES = [(28, 4, 128), (32, 4, 128), (40, 40, 128), (8, 8, 128), (16, 1, 64), (7, 1, 128),
           (14, 2, 128), (12, 6, 128), (2, 2, 64), (6, 2, 256)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(["rotary", "append8", "append8", "gather8", "decode8", "decode8", "varlen8",
                       "varlen8"])
    dtype = rng.choice(["bf16", "fp16"])
    hq, hkv, dim = rng.choice(_SHAPES)
    seed = rng.randrange(1 << 20)
    row = 2 * hkv * dim  # K and V values of a token in a layer
    if kind in ("rotary", "append8"):
        whole = rng.random() < 0.5
        seqs, mean = _log_int(rng, 1, 256), _log_int(rng, 4, 1024 if whole else 90)
        while seqs * (row + hq * dim) * (2 * mean if whole else BLOCK) > 32 << 20 and seqs > 1:
            seqs = (seqs + 1) // 2
        return _draw(kind, dtype, hq, hkv, dim, 1, seqs, mean, 0.5, 1, 2 * mean, seed,
                     whole=whole, rot=rng.choice([dim, dim, dim // 2]), inter=rng.random() < 0.5)
    if kind == "gather8":
        layers, seqs = rng.randint(1, 3), _log_int(rng, 1, 256)
        mean = _log_int(rng, 4, max(8, min(4096, (40 << 20) // (row * layers * seqs))))
        return _draw(kind, dtype, hq, hkv, dim, layers, seqs, mean, rng.choice([0.0, 0.8]), 1,
                     max(32, min(4 * mean, (60 << 20) // (row * layers * seqs))), seed)
    if kind == "decode8":
        layers = rng.randint(1, 4)
        seqs = _log_int(rng, 1, 512)
        mean = _log_int(rng, 8, max(16, min(65536, (500 << 20) // (row * layers * seqs))))
        return _draw(kind, dtype, hq, hkv, dim, layers, seqs, mean, rng.choice([0.0, 0.5, 1.0]),
                     1, max(32, min(131072, 6 * mean)), seed)
    if dim == 256:
        hq, hkv, dim = 28, 4, 128
    new = _log_int(rng, 1, 1500)
    seqs = _log_int(rng, 1, 64 if new < 64 else 8)
    top = int(2.0e11 / (4 * hq * dim * seqs * new))
    mean = max(new, _log_int(rng, 16, max(32, min(16384, top, (200 << 20) // (hkv * dim * seqs)))))
    return _draw(kind, dtype, hq, hkv, dim, 1, seqs, mean, rng.choice([0.0, 0.4, 0.8]), 1,
                 max(32, min(16384, 2 * mean)), seed, new=new, causal=rng.random() < 0.8)


def _draw(kind, *args, **more):
    c = _case("", kind, *args, **more)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(case):
    """The case's lengths (the same for every seed; prepare orders them by it)."""
    n, mean, sigma = case["seqs"], case["mean"], case["sigma"]
    if sigma == 0:
        return np.full(n, max(case["lo"], min(case["hi"], mean)), dtype=np.int64)
    rng = np.random.default_rng(case["lens_seed"])
    x = rng.lognormal(math.log(mean) - sigma * sigma / 2, sigma, size=n)
    return np.clip(np.rint(x), case["lo"], case["hi"]).astype(np.int64)


class State:
    """What the program holds: tensors and lists by name."""

    def __init__(self, **kw):
        self.__dict__.update(kw)


def _padded(tables):
    w = max(len(t) for t in tables)
    out = np.zeros((len(tables), w), dtype=np.int32)
    for i, t in enumerate(tables):
        out[i, :len(t)] = t
    return torch.from_numpy(out).cuda()


def _int32(x):
    return torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()


def _cumulated(x):
    return _int32(np.concatenate([[0], np.cumsum(x)]))


def _angles(positions, rot):
    """Cosines and sines of the rotation, float32 ``[positions, R]``."""
    freq = BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat([torch.cos(a), torch.sin(a)], 1).float()


def _row_bytes(hkv, dim):
    """Bytes of a layer's block of the 8-bit cache."""
    return 32 * hkv * dim + -(-4 * hkv // 128) * 128


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hkv, dim, layers = case["hq"], case["hkv"], case["dim"], case["layers"]
    kind = case["kind"]
    lens = rng.permutation(_lengths(case))
    n = len(lens)
    # channels of very different size, as projected keys have
    gain = torch.empty(hkv, dim, device="cuda").normal_(generator=gen).mul_(0.6).exp_()

    def rows(*shape):
        x = torch.empty(shape + (hkv, dim), device="cuda").normal_(generator=gen)
        return (x * gain).to(dt)

    need = [-(-int(x) // BLOCK) for x in lens]
    pool = int(sum(need) * 5 // 4) + 4
    ids = rng.permutation(pool)
    tables, o = [], 0
    for c in need:
        tables.append(ids[o:o + c].astype(np.int32).tolist())
        o += c
    st = State(kind=kind, dtype=dt, lens=lens, tables=tables, seq_lens=_int32(lens),
               longest=int(lens.max()), scale=1.0 / math.sqrt(dim), hq=hq, hkv=hkv, dim=dim)
    if kind == "rotary":
        st.cache = rows(pool, layers, 2, BLOCK)
    else:
        st.cache = torch.zeros((pool, layers, _row_bytes(hkv, dim)), dtype=torch.uint8,
                               device="cuda")
        # every block filled with rows that an append has written, a part at a time
        step = max(1, (1 << 25) // (layers * BLOCK * hkv * dim))
        for b in range(0, pool, step):
            m = min(step, pool - b)
            k, v = rows(m, layers, BLOCK), rows(m, layers, BLOCK)
            x = torch.stack([k, v], 3).float().permute(0, 1, 4, 3, 2, 5)  # [m, L, Hkv, 2, 16, D]
            _put(st.cache, slice(b, b + m), x, _exponent(x.abs().amax((-1, -2)), dt), dim)
    if kind in ("rotary", "append8"):
        at = [(b, p) for b, x in enumerate(lens)
              for p in (range(int(x)) if case["whole"] else [int(x) - 1])]
        st.slots = torch.tensor([tables[b][p // BLOCK] * BLOCK + p % BLOCK for b, p in at],
                                dtype=torch.int64, device="cuda")
        st.positions = torch.tensor([p for _, p in at], dtype=torch.int64, device="cuda")
        st.rot, st.inter = case["rot"], case["inter"]
        st.table = _angles(2 * case["hi"], st.rot)
        # the fused projection's output: queries, keys and values side by side
        qkv = torch.empty((len(at), (hq + 2 * hkv) * dim), device="cuda", dtype=dt)
        qkv.normal_(generator=gen)
        st.q, st.k, st.v = (x.unflatten(1, (-1, dim))
                            for x in qkv.split([hq * dim, hkv * dim, hkv * dim], 1))
        st.k.copy_(rows(len(at)))
        st.v.copy_(rows(len(at)))
        if not case["whole"]:  # read back: the blocks that the new tokens are in
            st.tables = [t[-1:] for t in tables]
            st.lens = (lens - 1) % BLOCK + 1
            st.seq_lens = _int32(st.lens)
            st.longest = int(st.lens.max())
    st.block_tables = _padded(st.tables)
    if kind in ("rotary", "append8", "gather8"):
        st.total = int(st.lens.sum())
        st.cu = _cumulated(st.lens)
        return st
    tokens = n
    if kind == "varlen8":
        st.new = np.minimum(lens, case["new"])
        st.causal = case["causal"]
        st.cu = _cumulated(st.new)
        st.most_new = int(st.new.max())
        tokens = int(st.new.sum())
    st.q = torch.empty((layers, tokens, hq, dim), device="cuda").normal_(generator=gen).to(dt)
    return st


# ---------------------------------------------------------------------------
# the operators' plain form
# ---------------------------------------------------------------------------
def _rotated(x, positions, table, inter):
    """Rows ``[T, H, D]`` turned by their positions' angles, float32."""
    half = table.size(1) // 2
    cos, sin = table[positions].unsqueeze(1).split(half, -1)  # [T, 1, R/2]
    f = x.float()
    a, b = (f[..., 0:2 * half:2], f[..., 1:2 * half:2]) if inter \
        else (f[..., :half], f[..., half:2 * half])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return torch.cat([turned, f[..., 2 * half:]], -1)


def _exponent(largest, dt):
    """The least e with ``largest <= 448 * 2^e``, within the type's bounds."""
    m, e = torch.frexp(largest)  # largest = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.where(largest == 0, torch.full_like(e, LOW[dt]), e).clamp(LOW[dt], TOP[dt])


def _power(e):
    """2^e of int32 exponents in the normal range, float32."""
    return ((e + 127) << 23).view(torch.float32)


def _codes(x, e):
    """Values ``[.., 16, D]`` (float32) -> code bytes under the exponents ``[..]``."""
    y = x * _power(-e)[..., None, None]
    y = torch.where(torch.isfinite(x), y.clamp(-LARGEST, LARGEST), torch.full_like(y, math.nan))
    return y.to(torch.float8_e4m3fn).view(torch.uint8)


def _code_views(blocks, hkv, dim):
    """K codes ``[.., H, chunk, token, dim]``, V codes ``[.., H, piece, quad,
    lane, dim, token]`` and the scale bytes ``[.., H, 4]`` of ``[.., R]`` bytes."""
    codes = blocks[..., :32 * hkv * dim].unflatten(-1, (hkv, 2, 16 * dim))
    return (codes[..., 0, :].unflatten(-1, (-1, 16, 16)),
            codes[..., 1, :].unflatten(-1, (-1, 4, 16, 4, 4)),
            blocks[..., 32 * hkv * dim:32 * hkv * dim + 4 * hkv].unflatten(-1, (hkv, 4)))


def _put(cache, at, x, e, dim):
    """Values ``[n, L, Hkv, 2, 16, D]`` under exponents ``[n, L, Hkv, 2]`` into
    the blocks ``at``."""
    c = _codes(x, e)
    new = cache[at].clone()
    k, v, s = _code_views(new, x.size(2), dim)
    k.copy_(c[..., 0, :, :].unflatten(-1, (-1, 16)).transpose(-3, -2))
    # [quad, token, lane, piece, dim] -> [piece, quad, lane, dim, token]
    lanes = c[..., 1, :, :].unflatten(-1, (16, -1, 4)).unflatten(-4, (4, 4))
    v.copy_(lanes.permute(*range(lanes.dim() - 5), -2, -5, -3, -1, -4))
    s[..., :2] = (e + 127).to(torch.uint8)
    cache[at] = new


def _values(blocks, hkv, dim):
    """Blocks ``[.., R]`` -> float32 values ``[.., Hkv, 2, 16, D]`` and
    exponents ``[.., Hkv, 2]``."""
    k, v, s = _code_views(blocks, hkv, dim)
    e = s[..., :2].to(torch.int32) - 127
    # [piece, quad, lane, dim, token] -> [quad, token, lane, piece, dim]
    v = v.permute(*range(v.dim() - 5), -4, -1, -3, -5, -2)
    c = torch.stack([k.transpose(-3, -2).flatten(-2), v.flatten(-3).flatten(-3, -2)], -3)
    f = c.contiguous().view(torch.float8_e4m3fn).float()
    return f * _power(e)[..., None, None], e


def _store(cache, key, value, slots, dt):
    """Rows ``[T, Hkv, D]`` (float32) into the slots of one layer ``[N, R]``."""
    hkv, dim = key.shape[1:]
    blocks, at = torch.unique(slots // BLOCK, return_inverse=True)
    off = slots % BLOCK
    first = torch.full_like(blocks, BLOCK).scatter_reduce_(0, at, off, "amin")
    x, e = _values(cache[blocks], hkv, dim)  # [n, Hkv, 2, 16, D], [n, Hkv, 2]
    new = torch.stack([key, value], 2)  # [T, Hkv, 2, D]
    largest = torch.zeros(e.shape, device="cuda")
    mine = torch.where(torch.isfinite(new), new.abs(), 0).amax(-1)
    largest.scatter_reduce_(0, at[:, None, None].expand_as(mine), mine, "amax")
    own_e = _exponent(largest, dt)
    e = torch.where((first == 0)[:, None, None], own_e, torch.maximum(e, own_e))
    # tokens of a block begun anew that none of these is have no meaning
    x = torch.where((first == 0)[:, None, None, None, None], torch.zeros_like(x), x)
    x[at, :, :, off] = new
    _put(cache.unsqueeze(1), blocks, x.unsqueeze(1), e.unsqueeze(1), dim)


def _padded_rows(st, layer):
    """K and V of a layer for every entry of the padded tables, float32
    ``[B, Hkv, width * 16, D]``."""
    ids = st.block_tables.long()
    x, _ = _values(st.cache[:, layer][ids], st.hkv, st.dim)  # [B, width, Hkv, 2, 16, D]
    return tuple(x[:, :, :, side].transpose(1, 2).flatten(2, 3) for side in (0, 1))


def _plain_rotary(st):
    q = _rotated(st.q, st.positions, st.table, st.inter).to(st.dtype)
    k = _rotated(st.k, st.positions, st.table, st.inter)
    if st.kind == "append8":
        _store(st.cache[:, 0], k, st.v.float(), st.slots, st.dtype)
        return {"q": q, **_plain_gather(st)}
    k = k.to(st.dtype)
    st.cache[st.slots // BLOCK, 0, 0, st.slots % BLOCK] = k
    st.cache[st.slots // BLOCK, 0, 1, st.slots % BLOCK] = st.v
    return {"q": q, "key": k, "cache": st.cache}


def _cached(st):
    """Which entries of the padded tables are tokens, ``[B, key]``."""
    return torch.arange(st.block_tables.size(1) * BLOCK, device="cuda") < st.seq_lens[:, None]


def _plain_gather(st):
    cached = _cached(st)
    sides = zip(*(_padded_rows(st, l) for l in range(st.cache.size(1))))
    k, v = (torch.stack([x.transpose(1, 2)[cached].to(st.dtype) for x in s]) for s in sides)
    return {"k": k, "v": v}


def _plain_attention(st):
    group = st.hq // st.hkv
    keys = torch.arange(st.block_tables.size(1) * BLOCK, device="cuda")
    if st.kind == "decode8":
        new, first = torch.ones_like(st.seq_lens), torch.arange(len(st.lens), device="cuda")
        most = 1
    else:
        new, first, most = st.cu[1:] - st.cu[:-1], st.cu[:-1].long(), st.most_new
    i = torch.arange(most, device="cuda")
    real = i < new[:, None]  # [B, query]
    at = torch.where(real, first[:, None] + i, 0)
    last = st.seq_lens[:, None] - 1 - torch.zeros_like(i)
    if st.kind == "varlen8" and st.causal:
        last = st.seq_lens[:, None] - new[:, None] + i
    hidden = (keys > last[..., None]).unsqueeze(1)  # [B, 1, query, key]

    def layer(l):
        k, v = _padded_rows(st, l)
        q = st.q[l][at].float().unflatten(2, (st.hkv, group)).permute(0, 2, 3, 1, 4)
        s = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)) * st.scale
        s = s.unflatten(2, (group, most))
        s.masked_fill_(hidden.unsqueeze(1), -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul((p / p.sum(-1, keepdim=True)).flatten(2, 3), v)
        o = o.unflatten(2, (group, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)
        return o[real].to(st.dtype)

    return {"out": [layer(l) for l in range(st.cache.size(1))]}


def _plain(st):
    if st.kind in ("rotary", "append8"):
        return _plain_rotary(st)
    if st.kind == "gather8":
        return _plain_gather(st)
    return _plain_attention(st)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    if not own:
        return _plain(st)
    from aegaeon_amd import attention as A
    from aegaeon_amd import kv8, rotary
    if st.kind == "rotary":
        key = torch.empty(st.k.shape, dtype=st.dtype, device="cuda")
        q = rotary.rotary_and_cache(st.q, st.k, st.v, st.cache[:, 0, 0], st.cache[:, 0, 1],
                                    st.slots, st.positions, st.table, interleaved=st.inter,
                                    out_key=key)
        return {"q": q, "key": key, "cache": st.cache}
    if st.kind in ("append8", "gather8"):
        out = {}
        if st.kind == "append8":
            out["q"] = kv8.rotary_and_cache_kv8(st.q, st.k, st.v, st.cache[:, 0], st.slots,
                                                st.positions, st.table, interleaved=st.inter)
        out["k"], out["v"] = kv8.gather_tokens_kv8(st.cache, st.block_tables, st.seq_lens,
                                                   st.total, st.longest, st.dim, dtype=st.dtype,
                                                   cu_seqlens=st.cu)
        return out
    if st.kind == "decode8":
        plan = A.DecodePlan(st.block_tables, st.seq_lens, st.longest, st.hkv)
        return {"out": [kv8.paged_decode_attention_kv8(st.q[l], st.cache[:, l], None, None,
                                                       st.scale, st.longest, plan=plan)
                        for l in range(st.cache.size(1))]}
    return {"out": [kv8.varlen_attention_kv8(st.q[l], st.cache[:, l], st.block_tables, st.cu,
                                             st.seq_lens, st.most_new, st.longest, st.scale,
                                             causal=st.causal)
                    for l in range(st.cache.size(1))]}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its outputs in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    hq, hkv, dim, layers = case["hq"], case["hkv"], case["dim"], case["layers"]
    lens = _lengths(case)
    n, total = len(lens), int(lens.sum())
    wide = 2 * hkv * dim * 2  # K and V of a token, 16 bits
    narrow = 2 * hkv * dim    # and as the 8-bit cache holds them
    blocks = int(sum(-(-int(x) // BLOCK) for x in lens))
    if case["kind"] in ("rotary", "append8"):
        new = total if case["whole"] else n
        places = int(lens.max()) if case["whole"] else len(set(lens.tolist()))
        # queries in and out, new rows in; slots, positions, the places' angles
        moved = new * (2 * hq * dim * 2 + wide + 16) + places * case["rot"] * 4
        if case["kind"] == "rotary":  # the rows, and the rotated keys once more
            return {"bytes": moved + new * (wide + wide // 2),
                    "flops": 3 * new * (hq + hkv) * case["rot"]}
        read = total if case["whole"] else int(((lens - 1) % BLOCK + 1).sum())
        touched = blocks if case["whole"] else n
        return {"bytes": moved + (new + read) * narrow + read * wide + 4 * touched * hkv
                + 4 * touched + 8 * n, "flops": 3 * new * (hq + hkv) * case["rot"]}
    if case["kind"] == "gather8":
        return {"bytes": layers * (total * (wide + narrow) + 2 * hkv * blocks) + 4 * blocks + 8 * n,
                "flops": 0}
    new = np.minimum(lens, case["new"]) if case["kind"] == "varlen8" else np.ones_like(lens)
    causal = case["kind"] == "varlen8" and case["causal"]
    pairs = int(sum(int(m) * int(x) - (int(m) * (int(m) - 1) // 2 if causal else 0)
                    for m, x in zip(new, lens)))
    return {"bytes": layers * (total * narrow + 2 * hkv * blocks
                               + 2 * int(new.sum()) * hq * dim * 2) + 4 * blocks + 4 * n,
            "flops": 4 * layers * hq * dim * pairs}


def _exact_rotated(x, positions, table, inter):
    """Rows ``[T, H, D]`` as complex numbers times their positions', in 64 bits."""
    half = table.size(1) // 2
    turn = torch.complex(table[positions, :half].double(), table[positions, half:].double())
    out = x.double().clone()
    first = slice(0, 2 * half, 2) if inter else slice(0, half)
    second = slice(1, 2 * half, 2) if inter else slice(half, 2 * half)
    z = torch.complex(out[..., first].contiguous(), out[..., second].contiguous()) * turn[:, None]
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _nearest(x, e):
    """x (64 bits) as the nearest code times 2^e."""
    y = (x.abs() * torch.exp2(-e)).clamp(max=LARGEST)
    # the step of y's binade: an eighth of its power of two, 2^-9 below 2^-6
    binade = torch.floor(torch.log2(y.clamp(min=2.0 ** -6)))
    binade = torch.where(torch.exp2(binade) > y, (binade - 1).clamp(min=-6), binade)
    binade = torch.where(torch.exp2(binade + 1) <= y, binade + 1, binade)
    step = torch.exp2(binade - 3)
    return torch.sign(x) * torch.round(y / step) * step * torch.exp2(e)


def _exact_exponent(a, dt):
    """The least e with a <= 448 * 2^e, from a logarithm corrected by trial."""
    e = torch.ceil(torch.log2(a.clamp(min=1e-300) / LARGEST))
    e = torch.where(a > LARGEST * torch.exp2(e), e + 1, e)
    e = torch.where(a <= LARGEST * torch.exp2(e - 1), e - 1, e)
    return e.clamp(LOW[dt], TOP[dt])


def _exact_block(layer, block, side, hkv, dim):
    """A block's K (side 0) or V (1) of a layer ``[N, R]`` in 64 bits, ``[16,
    Hkv, D]``, every value's byte looked up by its own address, and its
    exponents ``[Hkv]``; ``block [n]`` puts n in front of each."""
    t, d = torch.arange(BLOCK, device="cuda")[:, None], torch.arange(dim, device="cuda")[None, :]
    if side == 0:
        at = d // 16 * 256 + t * 16 + d % 16
    else:
        per = dim // 16
        at = ((d % per // 4 * 4 + t // 4) * 16 + d // per) * 16 + d % 4 * 4 + t % 4
    h = torch.arange(hkv, device="cuda")
    e = layer[block][:, 32 * hkv * dim + 4 * h + side].double() - 127
    c = layer[block][:, (2 * h[None, :, None] + side) * 16 * dim + at[:, None, :]].long()
    power, part = c // 8 % 16, c % 8
    x = torch.where(power == 0, part * 2.0 ** -9, (8 + part) * torch.exp2(power.double() - 10))
    return torch.where(c >= 128, -x, x) * torch.exp2(e)[:, None, :, None], e


def _exact_cached(st, layer, b, side):
    """Sequence b's K or V of a layer in 64 bits, ``[length, Hkv, D]``."""
    ids = torch.tensor(st.tables[b], device="cuda", dtype=torch.int64)
    x, _ = _exact_block(st.cache[:, layer], ids, side, st.hkv, st.dim)
    return x.flatten(0, 1)[:int(st.lens[b])]


def _exact_append(st):
    """What the sequences' listed blocks stand for once the new rows are in."""
    layer, out = st.cache[:, 0], {}
    new = (_exact_rotated(st.k, st.positions, st.table, st.inter), st.v.double())
    order = {int(s): i for i, s in enumerate(st.slots.tolist())}
    for side, name in enumerate(("k", "v")):
        parts = []
        for b, n in enumerate(st.lens):
            ids = torch.tensor(st.tables[b], device="cuda", dtype=torch.int64)
            x, e = _exact_block(layer, ids, side, st.hkv, st.dim)
            rows = [[order.get(i * BLOCK + t, -1) for t in range(BLOCK)] for i in st.tables[b]]
            rows = torch.tensor(rows, device="cuda")  # [blocks, 16]
            fresh = (rows[:, 0] >= 0)[:, None]
            joined = (rows >= 0)[..., None, None]
            mine = torch.where(joined, new[side][rows.clamp(min=0)], 0.0)
            own_e = _exact_exponent(mine.abs().amax((1, 3)), st.dtype)
            both = torch.where(fresh, own_e, torch.maximum(e, own_e))
            x = _nearest(torch.where(joined, mine, x), both[:, None, :, None])
            parts.append(x.flatten(0, 1)[:int(n)])
        out[name] = torch.cat(parts).unsqueeze(0)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    layers = st.cache.size(1)
    if st.kind in ("rotary", "append8"):
        q = _exact_rotated(st.q, st.positions, st.table, st.inter)
        if st.kind == "append8":
            return {"q": q, **_exact_append(st)}
        key, cache = _exact_rotated(st.k, st.positions, st.table, st.inter), st.cache.double()
        for side, x in ((0, key), (1, st.v.double())):
            cache[st.slots // BLOCK, 0, side, st.slots % BLOCK] = x
        return {"q": q, "key": key, "cache": cache}
    if st.kind == "gather8":
        k, v = (torch.stack([torch.cat([_exact_cached(st, l, b, side) for b in range(len(st.lens))])
                             for l in range(layers)]) for side in (0, 1))
        return {"k": k, "v": v}
    group = st.hq // st.hkv
    outs = []
    for l in range(layers):
        out = torch.zeros(st.q[l].shape, dtype=torch.float64, device="cuda")
        t = 0
        for b, n in enumerate(st.lens):
            n, m = int(n), int(st.new[b]) if st.kind == "varlen8" else 1
            k, v = _exact_cached(st, l, b, 0), _exact_cached(st, l, b, 1)
            keys = torch.arange(n, device="cuda")
            for h in range(st.hq):
                s = st.q[l, t:t + m, h].double() @ k[:, h // group].t().contiguous() * st.scale
                if st.kind == "varlen8" and st.causal:
                    s[keys[None, :] - (n - m) > torch.arange(m, device="cuda")[:, None]] = -math.inf
                out[t:t + m, h] = torch.softmax(s, -1) @ v[:, h // group].contiguous()
            t += m
        outs.append(out)
    return {"out": outs}

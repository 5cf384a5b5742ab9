"""The 4-bit KV cache's operators as measurable cases: the quantising append, the
de-page back to 16 bits, decode attention and the attention of several query
tokens per sequence, all over blocks of 16 tokens.

``listed`` names the cases, ``draw`` makes more of the same ranges, ``prepare``
makes what a program has in hand before the call, ``run`` is one pass (the
operators' plain form, or with ``own`` the framework's calls), ``work`` the
bytes and operations a pass cannot do without, ``exact`` the outputs in 64 bits.

The cache's numbers.  A group is 32 consecutive dims of one token's K or V row
of one head.  Its exponent e is the least integer with max|x| < 7 * 2^e, within
[-125, 125] (bf16) or [-125, 13] (fp16); a value's code is its sign and |x| / 2^e
rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code, at
most 6); the group keeps the byte e + 127.  A group that holds an infinity or a
NaN keeps 255 and stands for NaN.

The cache's bytes.  ``[N, L, Hkv, 2, R]`` uint8, a block's K and V records of a
layer and kv head, R = 8.5 D bytes: 8 D of codes (the lower dim of a pair in the
low half of its byte), then the scale bytes ``[D/32][16 tokens]``.  K codes are
``[chunk][16 tokens][min(16, D/8) bytes]``, a chunk's dims consecutive; V codes
``[piece][4 token quads][16 lanes][4 tokens][bytes]``, where lane j holds dims
D/16 j .. of a token, 8 (D 64: 4) per piece.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 16  # tokens per block
GROUP = 32  # dims per scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOP = {torch.bfloat16: 125, torch.float16: 13}  # largest exponent of a group
LOW = -125
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


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
        # A decode step's KV write for every layer at once (Qwen2.5-7B, 128
        # sequences), then the sequences' open blocks read back to 16 bits, as
        # an engine does that hands them to one with a 16-bit cache.
        _case("append_step_qwen_128", "append", "bf16", 28, 4, 128, 28, 128, 40, 0.5, 1, 96,
              whole=False),
        # A prompt run's KV write, eight layers of four 1024-token prompts, and
        # the rows it stands for read back for the prompt's own attention.
        _case("append_prompt_4x1024", "append", "bf16", 28, 4, 128, 8, 4, 1024, 0.0, 1, 1024,
              whole=True),
        # De-page of a batch of very different lengths, one layer.
        _case("gather_qwen_128", "gather", "bf16", 28, 4, 128, 1, 128, 400, 1.0, 16, 4096),
        # The same for a few short sequences of wide heads: latency.
        _case("gather_wide_6", "gather", "fp16", 6, 2, 256, 1, 6, 50, 0.8, 1, 128),
        # The smallest decode attention: one layer, eight short sequences.
        _case("decode_tiny", "decode", "fp16", 2, 2, 64, 1, 8, 60, 0.8, 1, 128),
        # A loaded engine: Qwen2.5-7B heads, 128 sequences of very different
        # lengths, one plan for the step's layers.
        _case("decode_qwen_128", "decode", "bf16", 28, 4, 128, 4, 128, 1500, 1.0, 16, 8192),
        # Multi-head attention without grouping (Llama-2-13B): the most cached
        # bytes per token, sequences of one length.
        _case("decode_llama_32", "decode", "fp16", 40, 40, 128, 1, 32, 2048, 0.0, 1, 4096),
        # One very long context: one sequence over the whole chip.
        _case("decode_long_context", "decode", "bf16", 28, 4, 128, 2, 1, 131001, 0.0, 1, 131072),
        # One kv head per GPU: Qwen2.5-7B cut over four GPUs by kv head.
        _case("decode_one_kv_head", "decode", "bf16", 7, 1, 128, 4, 256, 1000, 1.0, 16, 4096),
        # Five drafted tokens per sequence checked at once (Yi-1.5-9B heads).
        _case("varlen_draft_48", "varlen", "fp16", 32, 4, 128, 1, 48, 1000, 0.8, 16, 4096,
              new=5, causal=True),
        # The next chunks of four prompts over what is cached of them.
        _case("varlen_chunk_4x512", "varlen", "bf16", 28, 4, 128, 1, 4, 3800, 0.4, 600, 8192,
              new=512, causal=True),
        # The last chunk of one long document.
        _case("varlen_document", "varlen", "bf16", 28, 4, 128, 1, 1, 16001, 0.0, 1, 16384,
              new=2048, causal=True),
    ]


# (query heads, kv heads, head dim) of the framework's models and tests
_SHAPES = [(28, 4, 128), (32, 4, 128), (40, 40, 128), (8, 8, 128), (16, 1, 64), (7, 1, 128),
           (14, 2, 128), (12, 6, 128), (2, 2, 64), (6, 2, 256)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    kind = rng.choice(["append", "gather", "decode", "decode", "decode", "varlen", "varlen"])
    dtype = rng.choice(["bf16", "fp16"])
    hq, hkv, dim = rng.choice(_SHAPES)
    seed = rng.randrange(1 << 20)
    row = 2 * hkv * dim  # K and V values of a token in a layer
    if kind == "append":
        whole = rng.random() < 0.5
        layers, seqs = rng.choice([1, 8, 28]), _log_int(rng, 1, 256)
        mean = _log_int(rng, 4, 1024 if whole else 90)
        while seqs * layers * row * (2 * mean if whole else BLOCK) > 32 << 20 and seqs > 1:
            seqs = (seqs + 1) // 2
        while seqs * layers * row * (2 * mean if whole else BLOCK) > 32 << 20 and layers > 1:
            layers = (layers + 1) // 2
        return _draw(kind, dtype, hq, hkv, dim, layers, seqs, mean, 0.5, 1, 2 * mean, seed,
                     whole=whole)
    if kind == "gather":
        layers, seqs = rng.randint(1, 3), _log_int(rng, 1, 256)
        mean = _log_int(rng, 4, max(8, min(4096, (40 << 20) // (row * layers * seqs))))
        return _draw(kind, dtype, hq, hkv, dim, layers, seqs, mean, rng.choice([0.0, 0.8]), 1,
                     max(32, min(4 * mean, (60 << 20) // (row * layers * seqs))), seed)
    if kind == "decode":
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
    return _draw("varlen", dtype, hq, hkv, dim, 1, seqs, mean, rng.choice([0.0, 0.4, 0.8]), 1,
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
    cache = torch.zeros((pool, layers, hkv, 2, 17 * dim // 2), dtype=torch.uint8, device="cuda")
    # every block filled with rows that an append has written, a part at a time
    step = max(1, (1 << 25) // (layers * BLOCK * hkv * dim))
    for b in range(0, pool, step):
        m = min(step, pool - b)
        slots = torch.arange(b * BLOCK, (b + m) * BLOCK, device="cuda")
        _store(cache, rows(layers, m * BLOCK), rows(layers, m * BLOCK), slots)
    st = State(kind=kind, cache=cache, dtype=dt, lens=lens, tables=tables, seq_lens=_int32(lens),
               longest=int(lens.max()), scale=1.0 / math.sqrt(dim), hq=hq, hkv=hkv, dim=dim)
    if kind == "append":
        at = [(b, p) for b, x in enumerate(lens)
              for p in (range(int(x)) if case["whole"] else [int(x) - 1])]
        st.slots = torch.tensor([tables[b][p // BLOCK] * BLOCK + p % BLOCK for b, p in at],
                                dtype=torch.int64, device="cuda")
        st.k, st.v = rows(layers, len(at)), rows(layers, len(at))
        if not case["whole"]:  # read back: the blocks that the new tokens are in
            st.tables = [t[-1:] for t in tables]
            st.lens = (lens - 1) % BLOCK + 1
            st.seq_lens = _int32(st.lens)
            st.longest = int(st.lens.max())
    st.block_tables = _padded(st.tables)
    if kind in ("append", "gather"):
        st.total = int(st.lens.sum())
        st.cu = _cumulated(st.lens)
        return st
    tokens = n
    if kind == "varlen":
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
def _views(cache, dim):
    """The codes and scale bytes of a cache ``[..., Hkv, 2, R]``: K codes
    [..., chunk, token, byte], V codes [..., piece, quad, lane, token of the
    quad, byte] and both sides' scales [..., group, token]."""
    cb, w = min(16, dim // 8), min(8, dim // 16)
    k, v = cache[..., 0, :], cache[..., 1, :]
    return (k[..., :8 * dim].unflatten(-1, (-1, BLOCK, cb)),
            v[..., :8 * dim].unflatten(-1, (-1, 4, 16, 4, w // 2)),
            k[..., 8 * dim:].unflatten(-1, (-1, BLOCK)),
            v[..., 8 * dim:].unflatten(-1, (-1, BLOCK)))


def _quantise(x):
    """Rows ``[..., D]`` in 16 bits -> codes ``[..., D]`` and scale bytes
    ``[..., D/32]``."""
    f = x.float().unflatten(-1, (-1, GROUP))
    a = f.abs().amax(-1)
    finite = torch.isfinite(f).all(-1)
    m, e = torch.frexp(torch.where(finite, a, torch.ones_like(a)))
    e = torch.where(m < 0.875, e - 3, e - 2)  # m * 2^e < 0.875 * 2^(e' + 3)
    e = torch.where(a == 0, LOW, e.clamp(LOW, TOP[x.dtype]))
    # the reciprocal scale's bits: 2^-e is a normal number for every e
    y = f.abs() * ((127 - e) << 23).to(torch.int32).view(torch.float32).unsqueeze(-1)
    c = (y > 0.25).to(torch.uint8)
    for limit, ties in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True),
                        (5.0, False)):
        c += (y >= limit) if ties else (y > limit)
    c |= torch.signbit(f).to(torch.uint8) << 3
    c = torch.where(finite.unsqueeze(-1), c, torch.zeros_like(c))
    scales = torch.where(finite, e + 127, 255).to(torch.uint8)
    return c.flatten(-2), scales


def _packed(codes):
    """Two codes a byte, the lower dim in the low half."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _store(cache, key, value, slots):
    """Rows ``[L, T, Hkv, D]`` into the cache's slots."""
    dim = key.size(-1)
    kc, vc, ks, vs = _views(cache, dim)
    blk, off = slots // BLOCK, slots % BLOCK
    codes, scales = _quantise(key.transpose(0, 1))  # [T, L, Hkv, ..]
    kc[blk, :, :, :, off] = _packed(codes).unflatten(-1, (-1, kc.size(-1)))
    ks[blk, :, :, :, off] = scales
    codes, scales = _quantise(value.transpose(0, 1))
    # a row's bytes are [lane, piece, byte]
    vc[blk, :, :, :, off // 4, :, off % 4] = \
        _packed(codes).unflatten(-1, (16, vc.size(-5), vc.size(-1))).transpose(-2, -3)
    vs[blk, :, :, :, off] = scales


def _values(packed, scales):
    """Code bytes ``[..., D/2]`` and scale bytes ``[..., D/32]`` -> fp32."""
    grid = torch.tensor(GRID + tuple(-x for x in GRID), device=packed.device)
    c = torch.stack([packed & 15, packed >> 4], -1).flatten(-2)
    s = (scales.to(torch.int32) << 23).view(torch.float32)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (grid[c.int()].unflatten(-1, (-1, GROUP)) * s.unsqueeze(-1)).flatten(-2)


def _rows(blocks, dim):
    """K and V of blocks ``[n, Hkv, 2, R]`` as fp32 ``[Hkv, 16 n, D]``."""
    kc, vc, ks, vs = _views(blocks, dim)
    k = _values(kc.permute(1, 0, 3, 2, 4).flatten(-2), ks.permute(1, 0, 3, 2))
    # [n, Hkv, piece, quad, lane, token, byte] -> [Hkv, n, quad, token, lane, piece, byte]
    v = _values(vc.permute(1, 0, 3, 5, 4, 2, 6).flatten(-3).flatten(-3, -2),
                vs.permute(1, 0, 3, 2))
    return k.flatten(1, 2), v.flatten(1, 2)


def _padded_rows(st, layer):
    """K and V of a layer for every entry of the padded tables, fp32
    ``[B, Hkv, width * 16, D]``."""
    ids = st.block_tables.flatten().long()
    k, v = _rows(st.cache[:, layer].index_select(0, ids), st.dim)
    return (k.unflatten(1, (len(st.lens), -1)).transpose(0, 1),
            v.unflatten(1, (len(st.lens), -1)).transpose(0, 1))


def _plain(st):
    layers = range(st.cache.size(1))
    keys = torch.arange(st.block_tables.size(1) * BLOCK, device="cuda")
    cached = keys < st.seq_lens[:, None]  # [B, key]
    if st.kind in ("append", "gather"):
        if st.kind == "append":
            _store(st.cache, st.k, st.v, st.slots)
        sides = zip(*(_padded_rows(st, l) for l in layers))
        k, v = (torch.stack([x.transpose(1, 2)[cached].to(st.dtype) for x in s]) for s in sides)
        return {"k": k, "v": v}
    group = st.hq // st.hkv
    if st.kind == "decode":
        new, first = torch.ones_like(st.seq_lens), torch.arange(len(st.lens), device="cuda")
        most = 1
    else:
        new, first, most = st.cu[1:] - st.cu[:-1], st.cu[:-1].long(), st.most_new
    i = torch.arange(most, device="cuda")
    real = i < new[:, None]  # [B, query]
    at = torch.where(real, first[:, None] + i, 0)
    last = st.seq_lens[:, None] - 1 - torch.zeros_like(i)
    if st.kind == "varlen" and st.causal:
        last = st.seq_lens[:, None] - new[:, None] + i
    hidden = (keys > last[..., None]).unsqueeze(1)  # [B, 1, query, key]
    outs = []
    for l in layers:
        k, v = _padded_rows(st, l)
        q = st.q[l][at].float().unflatten(2, (st.hkv, group)).permute(0, 2, 3, 1, 4)
        s = torch.matmul(q.flatten(2, 3), k.transpose(2, 3)) * st.scale
        s = s.unflatten(2, (group, most))
        s.masked_fill_(hidden.unsqueeze(1), -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul((p / p.sum(-1, keepdim=True)).flatten(2, 3), v)
        o = o.unflatten(2, (group, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)
        outs.append(o[real].to(st.dtype))
    return {"out": outs}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    if not own:
        return _plain(st)
    from aegaeon_amd import attention as A
    from aegaeon_amd import kv4
    if st.kind in ("append", "gather"):
        if st.kind == "append":
            kv4.append_kv4(st.k, st.v, st.cache, st.slots)
        k, v = kv4.gather_tokens_kv4(st.cache, st.block_tables, st.seq_lens, st.total, st.longest,
                                     dtype=st.dtype, cu_seqlens=st.cu)
        return {"k": k, "v": v}
    outs = []
    if st.kind == "decode":
        plan = A.DecodePlan(st.block_tables, st.seq_lens, st.longest, st.hkv)
        for l in range(st.cache.size(1)):
            outs.append(kv4.paged_decode_attention_kv4(st.q[l], st.cache[:, l], None, None,
                                                       st.scale, st.longest, plan=plan))
        return {"out": outs}
    for l in range(st.cache.size(1)):
        outs.append(kv4.varlen_attention_kv4(st.q[l], st.cache[:, l], st.block_tables, st.cu,
                                             st.seq_lens, st.most_new, st.longest, st.scale,
                                             causal=st.causal))
    return {"out": outs}


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its outputs in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    hq, hkv, dim, layers = case["hq"], case["hkv"], case["dim"], case["layers"]
    lens = _lengths(case)
    n, total = len(lens), int(lens.sum())
    wide = 2 * hkv * dim * 2          # K and V of a token, 16 bits
    narrow = 2 * hkv * (dim * 17 // 32)  # and as the cache holds them
    blocks = int(sum(-(-int(x) // BLOCK) for x in lens))
    if case["kind"] == "append":
        new, read = (total, total) if case["whole"] else (n, int(((lens - 1) % BLOCK + 1).sum()))
        return {"bytes": layers * (new + read) * (wide + narrow) + 8 * new + 4 * n, "flops": 0}
    if case["kind"] == "gather":
        return {"bytes": layers * total * (wide + narrow) + 4 * blocks + 8 * n, "flops": 0}
    new = np.minimum(lens, case["new"]) if case["kind"] == "varlen" else np.ones_like(lens)
    causal = case["kind"] == "varlen" and case["causal"]
    pairs = int(sum(int(m) * int(x) - (int(m) * (int(m) - 1) // 2 if causal else 0)
                    for m, x in zip(new, lens)))
    return {"bytes": layers * (total * narrow + 2 * int(new.sum()) * hq * dim * 2) + 4 * blocks
            + 4 * n, "flops": 4 * layers * hq * dim * pairs}


def _exact_row_values(x):
    """What the rows ``[..., D]`` become in the cache, in 64 bits: the
    exponent from a logarithm and the nearest grid value by distance."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    flat, res = x.reshape(-1, GROUP), out.view(-1, GROUP)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    even = torch.arange(8, device=x.device) % 2  # of two equally near codes the even one
    for i in range(0, len(flat), 1 << 17):
        f = flat[i:i + (1 << 17)].double()
        a = f.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(a / 7)) + 1
        e = torch.where(a >= 7 * torch.exp2(e), e + 1, e)      # the logarithm's rounding
        e = torch.where(a < 7 * torch.exp2(e - 1), e - 1, e)
        e = torch.where(a == 0, torch.full_like(e, LOW), e.clamp(LOW, TOP[x.dtype]))
        y = (f.abs() * torch.exp2(-e)).unsqueeze(-1)
        d = (y - grid).abs()
        near = d == d.amin(-1, keepdim=True)
        pick = torch.where(near, even, torch.full_like(even, 9)).argmin(-1)
        res[i:i + (1 << 17)] = torch.sign(f) * grid[pick] * torch.exp2(e)
    return out


def _exact_cached(st, layer, b, side):
    """Sequence b's K (side 0) or V (1) of a layer in 64 bits, ``[length, Hkv,
    D]``: every value's byte looked up by its own address."""
    dim, n = st.dim, int(st.lens[b])
    t, d = torch.arange(n, device="cuda")[:, None], torch.arange(dim, device="cuda")[None, :]
    blk = torch.tensor(st.tables[b], device="cuda", dtype=torch.int64)[t // BLOCK]
    r = t % BLOCK
    if side == 0:
        cb = min(16, dim // 8)
        at = (d // (2 * cb) * BLOCK + r) * cb + d % (2 * cb) // 2
    else:
        per, w = dim // 16, min(8, dim // 16)
        lane, piece = d // per, d % per // w
        at = (((piece * 4 + r // 4) * 16 + lane) * 4 + r % 4) * (w // 2) + d % w // 2
    at, scale_at = at + 0 * d, 8 * dim + d // GROUP * BLOCK + r
    recs = st.cache[:, layer, :, side]  # [N, Hkv, R]
    out = []
    for h in range(st.hkv):
        byte = recs[blk, h, at].to(torch.int64)
        c = torch.where(d % 2 == 0, byte % 16, byte // 16)
        mag, e = c % 8, recs[blk, h, scale_at].double() - 127
        # a sign, two exponent bits and one of the mantissa
        x = torch.where(mag < 2, mag * 0.5,
                        (1 + (mag % 2) * 0.5) * torch.exp2((mag // 2 - 1).double()))
        out.append(torch.where(c >= 8, -x, x) * torch.exp2(e))
    return torch.stack(out, 1)


def exact(case, seed):
    st = prepare(case, seed)
    layers = st.cache.size(1)
    if st.kind in ("append", "gather"):
        sides = []
        for side in (0, 1):
            out = torch.zeros((layers, st.total, st.hkv, st.dim), dtype=torch.float64,
                              device="cuda")
            for l in range(layers):
                t = 0
                for b, n in enumerate(st.lens):
                    if st.kind == "gather" or not case["whole"]:
                        out[l, t:t + int(n)] = _exact_cached(st, l, b, side)
                    t += int(n)
            if st.kind == "append":
                new = _exact_row_values((st.k, st.v)[side])
                if case["whole"]:
                    out = new
                else:
                    out[:, st.cu[1:].long() - 1] = new
            sides.append(out)
        return {"k": sides[0], "v": sides[1]}
    group = st.hq // st.hkv
    outs = []
    for l in range(layers):
        out = torch.zeros(st.q[l].shape, dtype=torch.float64, device="cuda")
        t = 0
        for b, n in enumerate(st.lens):
            n, m = int(n), int(st.new[b]) if st.kind == "varlen" else 1
            k, v = _exact_cached(st, l, b, 0), _exact_cached(st, l, b, 1)
            keys = torch.arange(n, device="cuda")
            for h in range(st.hq):
                s = st.q[l, t:t + m, h].double() @ k[:, h // group].t().contiguous() * st.scale
                if st.kind == "varlen" and st.causal:
                    s[keys[None, :] - (n - m) > torch.arange(m, device="cuda")[:, None]] = -math.inf
                out[t:t + m, h] = torch.softmax(s, -1) @ v[:, h // group].contiguous()
            t += m
        outs.append(out)
    return {"out": outs}

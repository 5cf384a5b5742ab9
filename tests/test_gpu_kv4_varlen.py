"""GPU parity of the attention of several query tokens per sequence over the
4-bit KV cache with the oracle's float64 textbook over the stored values.

The stored values are exact in 16 bits and the arithmetic past them is the
prompt attention's (fp32 scores, P rounded to 16 bits before P.V), so the bars
are test_gpu_prefill.py's: the relative L2 error of the float64 result rounded to
the output type plus 1e-3 (bf16) / 1.5e-4 (fp16) for P's rounding, and per
element 2^-7 / 2^-9 of the output's largest magnitude."""
import math
import threading

import numpy as np
import pytest
import torch

from aegaeon_amd import attention as A
from aegaeon_amd import kv4
from aegaeon_amd._lib import AegkvError
from oracle import kv4_oracle as k4
from oracle import kv_oracle as ko
from tests.kvtest_utils import random_bits, to_device_bits

pytestmark = pytest.mark.gpu

BARS = {"bf16": (1e-3, 2.0 ** -7), "fp16": (1.5e-4, 2.0 ** -9)}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


class Batch:
    """New and cached tokens per sequence, a filled cache with stale bytes
    behind the last tokens, queries; on both sides."""

    def __init__(self, device, new, lens, Hq, Hkv, D, dtype, seed, extra=0, spare=2):
        rng = self.rng = np.random.default_rng(seed)
        self.new, self.lens = np.asarray(new), np.asarray(lens)
        self.Hq, self.Hkv, self.D, self.dtype = Hq, Hkv, D, dtype
        need = [-(-int(x) // 16) for x in lens]
        n = sum(need) + spare
        ids = [int(x) for x in rng.permutation(n)]
        self.tables = [[ids.pop() for _ in range(c)] for c in need]
        gain = np.exp(0.5 * rng.standard_normal(D))
        x = ko.bits_to_float(random_bits(rng, (2, 1, n * 16, Hkv, D), dtype), dtype) * gain
        x = ko.bits_to_float(ko.float_to_bits(x, dtype), dtype)
        cache = np.zeros((n, 1, Hkv, 2, k4.record_bytes(D)), dtype=np.uint8)
        k4.append(x[0], x[1], cache, np.arange(n * 16), dtype)
        self.cache = cache[:, 0]
        for t, x in zip(self.tables, self.lens):
            for r in range(x % 16, 16) if x % 16 else ():
                self.cache[t[-1], :, :, 8 * D + r::16] = 255
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.q = random_bits(rng, (int(self.cu[-1]) + extra, Hq, D), dtype)
        self.dq = to_device_bits(self.q, dtype, device)
        self.dc = torch.from_numpy(self.cache).to(device)
        self.bt = torch.from_numpy(ko.pad_block_tables(self.tables)).to(device)
        self.dcu = torch.from_numpy(self.cu).to(device)
        self.sl = torch.from_numpy(self.lens.astype(np.int32)).to(device)

    def run(self, scale, causal=True, max_q=None, max_len=None, **kw):
        return kv4.varlen_attention_kv4(
            kw.pop("q", self.dq), kw.pop("cache", self.dc), self.bt, self.dcu, self.sl,
            int(max(self.new)) if max_q is None else max_q,
            int(max(self.lens)) if max_len is None else max_len, scale, causal=causal, **kw)

    def want(self, scale, causal=True):
        k, v = (np.nan_to_num(x) for x in k4.rows(self.cache, self.D))
        return k4.varlen_attention(ko.bits_to_float(self.q, self.dtype), k, v, self.tables,
                                   self.cu, self.lens, scale, causal)

    def check(self, out, scale, causal=True):
        within(out.double().cpu().numpy(), self.want(scale, causal), self.dtype)


def within(got, ref, dtype):
    assert np.isfinite(got).all()
    extra, elem = BARS[dtype]
    norm = max(np.linalg.norm(ref), 1e-30)
    err = np.linalg.norm(got - ref) / norm
    rounding = np.linalg.norm(torch.from_numpy(ref).to(DTYPES[dtype]).double().numpy() - ref) / norm
    assert err <= rounding + extra, (err, rounding)
    worst = np.abs(got - ref).max() / max(np.abs(ref).max(), 1e-30)
    assert worst <= elem, worst


NEW = [1, 5, 0, 16, 33, 64, 129, 7, 300]
LENS = [1, 200, 40, 16, 97, 64, 700, 1031, 300]


@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (8, 8, 64), (16, 1, 128), (12, 3, 64),
                                      (40, 2, 128)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_ragged_batch(device, Hq, Hkv, D, causal, dtype):
    b = Batch(device, NEW, LENS, Hq, Hkv, D, dtype, Hq + D)
    scale = 1 / math.sqrt(D)
    b.check(b.run(scale, causal), scale, causal)


@pytest.mark.parametrize("new,lens", [
    ([1], [1]), ([1], [63]), ([1], [64]), ([1], [65]), ([1] * 5, [5000, 3, 16, 17, 2049]),
    ([2048], [2048]), ([1500, 3], [1500, 9000]), ([700], [701]), ([257], [4000]),
    ([4] * 70, list(range(4, 74)))])
@pytest.mark.parametrize("Hq,Hkv,D", [(14, 2, 128), (4, 4, 64)])
def test_lengths(device, new, lens, Hq, Hkv, D):
    """One token, chunks that are the whole prompt, short chunks over long
    caches (cut over workgroups), long ones."""
    b = Batch(device, new, lens, Hq, Hkv, D, "bf16", len(new) + sum(lens))
    b.check(b.run(0.1), 0.1)


@pytest.mark.parametrize("new,lens,Hq,Hkv,D", [
    ([1200], [2500], 14, 2, 128),                      # four waves, one key tile per step
    ([200] * 9, [1000] * 9, 8, 8, 64),
    ([64] * 40, [5000] + [100] * 39, 8, 8, 64),        # two, one sequence cut of many
    ([64] * 140, [70] * 139 + [5000], 8, 8, 64),       # of very many
    ([300] * 140, [6000] + [300] * 139, 2, 2, 64)])
def test_cut_sequences_of_many_rows(device, new, lens, Hq, Hkv, D):
    b = Batch(device, new, lens, Hq, Hkv, D, "bf16", sum(lens))
    b.check(b.run(0.1), 0.1)


# Few tiles of many rows and keys: eight-wave workgroups, whole (47 tiles of 256
# rows and more per kv head) and cut.
@pytest.mark.parametrize("new,lens", [([1, 300, 700], [50, 5000, 6200]), ([600], [6001]),
                                      ([40, 300], [2000, 9600])])
@pytest.mark.parametrize("dtype,causal", [("bf16", True), ("fp16", False)])
def test_few_tiles_of_many_keys(device, new, lens, dtype, causal):
    b = Batch(device, new, lens, 40, 2, 128, dtype, sum(lens))
    b.check(b.run(-0.1, causal), -0.1, causal)


def test_nan_and_unreadable_blocks_of_long_rows(device):
    """As the tests below for fewer rows: a NaN of V shows in its dims of the rows
    that attend to its token, and an unreadable block is masked."""
    b = Batch(device, [600], [6001], 40, 2, 128, "bf16", 3)
    token, grp = 5700, 2
    dirty = b.dc.clone()
    dirty[b.tables[0][token // 16], 1, 1, 8 * 128 + grp * 16 + token % 16] = 255
    clean, out = b.run(0.1), b.run(0.1, cache=dirty)
    seen = torch.zeros(out.shape, dtype=torch.bool, device=device)
    seen[token - 5401:, 20:, 32 * grp:32 * grp + 32] = True
    assert torch.isnan(out[seen].float()).all()
    assert torch.equal(out[~seen].view(torch.int16), clean[~seen].view(torch.int16))
    bad = b.bt.clone()
    bad[0, token // 16] = b.dc.size(0)
    gone = kv4.varlen_attention_kv4(b.dq, dirty, bad, b.dcu, b.sl, 600, 6001, 0.1)
    k, v = (np.nan_to_num(x) for x in k4.rows(b.cache, 128))
    rows = [np.ascontiguousarray(x[b.tables[0]].reshape(-1, 2, 128)[:6001].swapaxes(0, 1))
            for x in (k, v)]
    keep = np.arange(6001) // 16 != token // 16
    q = ko.bits_to_float(b.q, "bf16")
    want = np.zeros(q.shape)
    for h in range(40):
        s = np.ascontiguousarray(q[:, h]) @ rows[0][h // 20].T * 0.1
        s[~(keep & (np.arange(6001) <= 5401 + np.arange(600)[:, None]))] = -np.inf
        p = np.exp(s - s.max(-1, keepdims=True))
        want[:, h] = p @ rows[1][h // 20] / p.sum(-1, keepdims=True)
    within(gone.double().cpu().numpy(), want, "bf16")


@pytest.mark.parametrize("first", [1, 100, 300])
def test_more_sequences_than_threads(device, first):
    new = [first] + [1, 0, 2] * 400
    b = Batch(device, new, [2000] + [3, 40, 17] * 400, 2, 1, 64, "bf16", first)
    b.check(b.run(0.1), 0.1)


def test_threads_share_a_stream(device):
    sets = [Batch(device, [5, 40], [3000, 700], 28, 4, 128, "bf16", 11),
            Batch(device, [300], [2500], 14, 2, 128, "bf16", 12)]
    want = [b.run(0.1) for b in sets]
    got = [[], []]

    def calls(i):
        for _ in range(20):
            got[i].append(sets[i].run(0.1))

    threads = [threading.Thread(target=calls, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs, w in zip(got, want):
        assert len(outs) == 20
        assert all(torch.equal(o.view(torch.int16), w.view(torch.int16)) for o in outs)


def test_one_query_is_the_decode_attention(device):
    lens = [1, 77, 1024, 3000]
    b = Batch(device, [1] * 4, lens, 28, 4, 128, "fp16", 8)
    out = b.run(0.09)
    dec = kv4.paged_decode_attention_kv4(b.dq, b.dc, b.bt, b.sl, 0.09, 3000)
    b.check(out, 0.09)
    b.check(dec, 0.09)


def test_queries_before_the_first_key(device):
    """Fewer cached tokens than queries: the first queries see nothing and
    give zeros; a sequence without a cached token gives zeros throughout."""
    new, lens = [40, 8, 5], [10, 0, 5]
    b = Batch(device, new, lens, 8, 2, 128, "bf16", 3)
    out = b.run(0.1)
    assert not out[:30].any() and not out[40:48].any()
    b.check(out, 0.1)
    b.check(b.run(0.1, causal=False), 0.1, causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.1, 2.0])
def test_scales(device, scale):
    b = Batch(device, [70, 3], [300, 90], 8, 2, 128, "bf16", 4)
    b.check(b.run(scale), scale)


def test_strides_bounds_and_rows_left_alone(device):
    """Queries that are columns of a fused projection, an output inside a
    wider buffer, a layer of a larger cache, tokens behind the last sequence and
    past max_seqlen_q left as they were, keys past max_seq_len not attended."""
    Hq, Hkv, D = 14, 2, 128
    b = Batch(device, [20, 90], [50, 400], Hq, Hkv, D, "bf16", 12, extra=6)
    T = b.q.shape[0]
    fused = torch.zeros(T, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device=device)
    fused[:, :Hq * D] = b.dq.flatten(1)
    wide = torch.full((T, Hq * D + 16), 3.0, dtype=torch.bfloat16, device=device)
    layers = torch.full((b.dc.size(0), 3, Hkv, 2, 1088), 255, dtype=torch.uint8, device=device)
    layers[:, 2] = b.dc
    out = wide[:, :Hq * D].unflatten(1, (Hq, D))
    b.run(0.1, q=fused[:, :Hq * D].unflatten(1, (Hq, D)), cache=layers[:, 2], out=out)
    assert bool((wide[:, Hq * D:] == 3.0).all()) and bool((wide[110:] == 3.0).all())
    within(out[:110].double().cpu().numpy(), b.want(0.1)[:110], "bf16")
    out2 = torch.full_like(b.dq, 7.0)
    b.run(0.1, max_q=32, out=out2)
    # (another bound, another cut of the keys: other last bits)
    within(out2[:52].double().cpu().numpy(), b.want(0.1)[:52], "bf16")
    assert bool((out2[52:] == 7.0).all())
    # the bound of the keys: 64 of sequence 1's 400, whose queries come later
    out3 = b.run(0.1, max_len=64, causal=True)
    k, v = (np.nan_to_num(x) for x in k4.rows(b.cache, D))
    want = k4.varlen_attention(ko.bits_to_float(b.q, "bf16"), k, v, b.tables, b.cu, [50, 64], 0.1,
                               False)
    within(out3[20:110].double().cpu().numpy(), want[20:110], "bf16")


def test_unreadable_blocks_are_masked(device):
    b = Batch(device, [5, 40], [300, 200], 8, 2, 64, "bf16", 17)
    bad = b.bt.clone()
    bad[0, 3], bad[0, 0], bad[1, 2] = b.dc.size(0), -7, 1 << 30
    out = kv4.varlen_attention_kv4(b.dq, b.dc, bad, b.dcu, b.sl, 40, 300, 0.1)
    k, v = (np.nan_to_num(x) for x in k4.rows(b.cache, 64))
    q = ko.bits_to_float(b.q, "bf16")
    want = np.zeros(q.shape)
    for s, gone in ((0, (3, 0)), (1, (2,))):
        n, m, t0 = int(b.lens[s]), int(b.new[s]), int(b.cu[s])
        keep = np.array([j // 16 not in gone for j in range(n)])
        kk, vv = k[b.tables[s]].reshape(-1, 2, 64)[:n], v[b.tables[s]].reshape(-1, 2, 64)[:n]
        for i in range(m):
            see = keep & (np.arange(n) <= n - m + i)
            for h in range(8):
                x = kk[see, h // 4] @ q[t0 + i, h] * 0.1
                p = np.exp(x - x.max())
                want[t0 + i, h] = p @ vv[see, h // 4] / p.sum()
    within(out.double().cpu().numpy(), want, "bf16")


@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("token,lens", [(130, [160]), (150, [160]), (159, [160]), (20, [2000])])
def test_a_nan_shows_where_its_token_is_attended_and_nowhere_else(device, side, D, token, lens):
    """One group of one token NaN (its codes arbitrary): K spoils the rows that
    see it in its head, V their dims of that group; the others keep their bits."""
    b = Batch(device, [30], lens, 4, 2, D, "bf16", 9)
    clean = b.run(0.1)
    blk, r, grp = b.tables[0][token // 16], token % 16, D // 32 - 1
    dirty = b.dc.clone()
    dirty[blk, 1, side, 8 * D + grp * 16 + r] = 255
    out = b.run(0.1, cache=dirty)
    first = token - (lens[0] - 30)  # the first query that sees it
    seen = torch.zeros(out.shape, dtype=torch.bool, device=device)
    seen[max(first, 0):, 2:, (32 * grp if side else 0):] = True
    assert torch.isnan(out[seen].float()).all()
    assert torch.equal(out[~seen].view(torch.int16), clean[~seen].view(torch.int16))


def test_captured_calls_share_nothing(device):
    sets = [Batch(device, [5, 40], [3000, 700], 28, 4, 128, "bf16", s) for s in (1, 2)]
    outs = [torch.empty_like(b.dq) for b in sets]
    side, graphs = torch.cuda.Stream(), []
    for b, o in zip(sets, outs):
        b.run(0.1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            b.run(0.1, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for b in sets:
            b.dq.mul_(-1.5)
        want = [b.run(0.1) for b in sets]
        torch.cuda.synchronize()
        for _ in range(3):
            for st, g in zip(streams, graphs):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o.view(torch.int16), w.view(torch.int16))


def test_a_callers_workspace_and_repeated_calls_give_the_same_bits(device):
    b = Batch(device, [5, 40, 8], [3000, 700, 90], 28, 4, 128, "bf16", 5)
    ws = kv4.varlen_attention_workspace(3, 53, 40, 3000, 28, 4, 128)
    first = b.run(0.1)
    for _ in range(3):
        ws.fill_(0xFF)
        assert torch.equal(b.run(0.1, workspace=ws).view(torch.int16), first.view(torch.int16))
    with pytest.raises(ValueError, match="workspace"):
        b.run(0.1, workspace=ws[:-1])


def test_a_chunked_prompt_gives_the_whole_ones_rows(device):
    """A prompt appended and attended chunk by chunk, in one call, by the
    16-bit prompt attention over the de-paged rows, and its last token by the
    decode attention: each within its bars of the textbook."""
    Hq, Hkv, D, n = 28, 4, 128, 500
    rng = np.random.default_rng(31)
    cache = kv4.kv4_cache(40, 1, Hkv, D, device)
    table = [int(x) for x in rng.permutation(40)[:-(-n // 16)]]
    slots = torch.tensor([table[p // 16] * 16 + p % 16 for p in range(n)], device=device)
    qkv = to_device_bits(random_bits(rng, (n, (Hq + 2 * Hkv) * D), "bf16"), "bf16", device)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    bt = torch.tensor([table], dtype=torch.int32, device=device)
    parts, at = [], 0
    for m in (200, 1, 130, 169):
        kv4.reshape_and_cache_kv4(k[at:at + m], v[at:at + m], cache[:, 0], slots[at:at + m])
        at += m
        parts.append(kv4.varlen_attention_kv4(
            q[at - m:at], cache[:, 0], bt, torch.tensor([0, m], dtype=torch.int32, device=device),
            torch.tensor([at], dtype=torch.int32, device=device), m, at, 0.09))
    cu = torch.tensor([0, n], dtype=torch.int32, device=device)
    whole = kv4.varlen_attention_kv4(q, cache[:, 0], bt, cu, cu[1:], n, n, 0.09)
    gk, gv = kv4.gather_tokens_kv4(cache, bt, cu[1:], n, n)
    prompt = A.varlen_prefill_attention(q, gk[0], gv[0], cu, n, 0.09)
    last = kv4.paged_decode_attention_kv4(q[-1:], cache[:, 0], bt, cu[1:], 0.09, n)
    rows = [np.stack([k4.decode(*k4.encode(x.double().cpu().numpy(), "bf16"))]) for x in (k, v)]
    pad = [np.concatenate([x[0], np.zeros((-n % 16, Hkv, D))]).reshape(-1, 16, Hkv, D) for x in rows]
    want = k4.varlen_attention(q.double().cpu().numpy(), *pad, [list(range(len(table)))], [0, n],
                               [n], 0.09, True)
    for got in (torch.cat(parts), whole, prompt):
        within(got.double().cpu().numpy(), want, "bf16")
    within(last.double().cpu().numpy(), want[-1:], "bf16")


def test_refusals(device):
    b = Batch(device, [3], [40], 8, 2, 128, "bf16", 1)
    with pytest.raises(ValueError, match="cu_seqlens_q"):
        kv4.varlen_attention_kv4(b.dq, b.dc, b.bt, b.dcu.long(), b.sl, 3, 40, 0.1)
    with pytest.raises(ValueError, match="block_tables"):
        kv4.varlen_attention_kv4(b.dq, b.dc, b.bt[0], b.dcu, b.sl, 3, 40, 0.1)
    with pytest.raises(ValueError, match="kv_cache"):
        kv4.varlen_attention_kv4(b.dq, b.dc[:, :, :, :544], b.bt, b.dcu, b.sl, 3, 40, 0.1)
    with pytest.raises(ValueError, match="out"):
        b.run(0.1, out=torch.empty_like(b.dq).half())
    with pytest.raises(AegkvError):  # 100 keys need more blocks than the table has
        b.run(0.1, max_len=100)
    with pytest.raises(AegkvError):
        b.run(float("nan"))
    with pytest.raises(AegkvError):
        kv4.varlen_attention_kv4(b.dq[:, :7], b.dc, b.bt, b.dcu, b.sl, 3, 40, 0.1)  # 7 over 2
    c256 = kv4.kv4_cache(4, 1, 2, 256, device)
    with pytest.raises(AegkvError):
        kv4.varlen_attention_kv4(torch.zeros(3, 8, 256, dtype=torch.bfloat16, device=device),
                                 c256[:, 0], b.bt, b.dcu, b.sl, 3, 16, 0.1)
    for t in (b.dc, b.bt, b.dcu, b.sl):
        assert t.is_cuda
    with pytest.raises(ValueError, match="seq_lens"):
        kv4.varlen_attention_kv4(b.dq, b.dc, b.bt, b.dcu, b.sl.cpu(), 3, 40, 0.1)
    empty = kv4.varlen_attention_kv4(b.dq[:0], b.dc, b.bt, b.dcu, b.sl, 3, 40, 0.1)
    assert empty.shape == (0, 8, 128)

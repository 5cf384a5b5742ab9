"""GPU parity of the 4-bit KV cache (append, de-page, decode attention) with
the oracle.

Append and de-page are exact: every byte of the cache and every 16-bit value.
Decode attention does the 16-bit cache's arithmetic on the stored values, which
are exact in 16 bits, so its bars are those of test_gpu_attention.py: 2e-3
relative L2, and per element one ulp of the output type plus 1e-5 and 2^-17 of
the largest |v| (each softmax weight keeps 16 significant bits)."""
import math

import numpy as np
import pytest
import torch

from aegaeon_amd import attention as A
from aegaeon_amd import kv4, ops
from aegaeon_amd._lib import AegkvError
from oracle import kv4_oracle as k4
from oracle import kv_oracle as ko
from tests.kvtest_utils import bf16_ulp, fp16_ulp, random_bits, to_bits, to_device_bits

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _poisoned(n, layers, heads, dim):
    return np.full((n, layers, heads, 2, k4.record_bytes(dim)), 0xFF, dtype=np.uint8)


def _append(device, key, value, cache, slots, dtype):
    """Both sides append the same rows (uint16 bits [L, T, Hkv, D])."""
    dev = torch.from_numpy(cache).to(device)
    kv4.append_kv4(to_device_bits(key, dtype, device), to_device_bits(value, dtype, device), dev,
                   torch.from_numpy(slots).to(device))
    k4.append(ko.bits_to_float(key, dtype), ko.bits_to_float(value, dtype), cache, slots, dtype)
    return dev


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("L,H,D", [(1, 1, 64), (3, 4, 128), (2, 3, 256), (2, 5, 64)])
@pytest.mark.parametrize("T", [1, 7, 50])
def test_append_bytes(device, dtype, L, H, D, T):
    """Random slots, some negative and some past the pool: the whole cache
    equals the oracle's, untouched bytes included."""
    rng = np.random.default_rng(L * 100 + D + T)
    cache = _poisoned(5, L, H, D)
    slots = rng.permutation(5 * 16)[:T].astype(np.int64)
    if T > 3:
        slots[1], slots[T // 2] = -1, 5 * 16
    k, v = random_bits(rng, (L, T, H, D), dtype), random_bits(rng, (L, T, H, D), dtype)
    dev = _append(device, k, v, cache, slots, dtype)
    assert np.array_equal(dev.cpu().numpy(), cache)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("order", ["sorted", "mixed"])
def test_append_of_every_16_bit_pattern(device, dtype, D, order):
    """All 65536 patterns: zeros, subnormals, infinities and NaN among them, in
    groups of like magnitude and in groups of any."""
    bits = np.arange(1 << 16, dtype=np.uint16)
    if order == "mixed":
        # each half's magnitudes rise together, so a group is of one kind in
        # two signs; then a shuffle within windows of 4096 patterns
        rng = np.random.default_rng(5)
        bits = bits.reshape(16, 4096)
        bits = np.stack([rng.permutation(x) for x in bits]).reshape(-1)
    T = (1 << 16) // D
    k = bits.reshape(1, T, 1, D).copy()
    v = k[:, ::-1].copy()
    cache = _poisoned(T // 16 + 1, 1, 1, D)
    dev = _append(device, k, v, cache, np.arange(T, dtype=np.int64) + 3, dtype)
    assert np.array_equal(dev.cpu().numpy(), cache)


def test_append_strided_rows_and_layer_view(device):
    """Rows that are slices of a fused projection, one layer of a cache of
    several: the other layers' bytes stay."""
    rng = np.random.default_rng(8)
    T, H, D = 37, 4, 128
    fused = random_bits(rng, (T, 12 * D), "bf16")
    dev_fused = to_device_bits(fused, "bf16", device)
    key = dev_fused[:, 4 * D:8 * D].unflatten(1, (H, D))
    value = dev_fused[:, 8 * D:].unflatten(1, (H, D))
    cache = _poisoned(6, 3, H, D)
    dev = torch.from_numpy(cache).to(device)
    slots = rng.permutation(96)[:T].astype(np.int64)
    kv4.reshape_and_cache_kv4(key, value, dev[:, 1], torch.from_numpy(slots).to(device))
    f = ko.bits_to_float(fused, "bf16")
    k4.append(f[None, :, 4 * D:8 * D].reshape(1, T, H, D), f[None, :, 8 * D:].reshape(1, T, H, D),
              cache[:, 1:2], slots, "bf16")
    assert np.array_equal(dev.cpu().numpy(), cache)


def test_append_of_no_tokens(device):
    cache = torch.full((2, 1, 2, 2, 544), 7, dtype=torch.uint8, device=device)
    x = torch.empty(1, 0, 2, 64, dtype=torch.float16, device=device)
    kv4.append_kv4(x, x, cache, torch.empty(0, dtype=torch.int64, device=device))
    assert bool((cache == 7).all())


# ---------------------------------------------------------------------------
# de-page
# ---------------------------------------------------------------------------
def _filled(rng, n, layers, heads, dim, dtype):
    """A cache whose every slot was written, as the oracle holds it."""
    cache = _poisoned(n, layers, heads, dim)
    x = rng.standard_normal((2, layers, n * 16, heads, dim)) * np.exp(rng.standard_normal(dim))
    x = ko.bits_to_float(ko.float_to_bits(x, dtype), dtype)
    k4.append(x[0], x[1], cache, np.arange(n * 16), dtype)
    return cache


def _tables(rng, lens, pool):
    need = [-(-int(x) // 16) for x in lens]
    ids = rng.permutation(pool)
    out, o = [], 0
    for c in need:
        out.append([int(x) for x in ids[o:o + c]])
        o += c
    return out


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("H,D", [(1, 64), (4, 128), (2, 256), (11, 128)])
def test_gather_values(device, dtype, H, D):
    rng = np.random.default_rng(H + D)
    lens = np.array([1, 0, 15, 16, 17, 70, 33])
    cache = _filled(rng, 24, 3, H, D, dtype)
    tables = _tables(rng, lens, 24)
    padded = ko.pad_block_tables(tables)
    for layers in (None, (1, 2)):
        k, v = kv4.gather_tokens_kv4(torch.from_numpy(cache).to(device),
                                     torch.from_numpy(padded).to(device),
                                     torch.from_numpy(lens.astype(np.int32)).to(device),
                                     int(lens.sum()), int(lens.max()), dtype=DTYPES[dtype],
                                     layers=layers)
        first, count = layers or (0, 3)
        for l in range(count):
            rows = k4.rows(cache[:, first + l], D)
            for got, side in ((k, rows[0]), (v, rows[1])):
                want = np.concatenate([side[t].reshape(-1, H, D)[:n] if t else side[:0].reshape(0, H, D)
                                       for t, n in zip(tables, lens)])
                assert np.array_equal(got[l].double().cpu().numpy(), want)


def test_gather_leaves_what_it_is_not_to_write(device):
    """Gaps between the sequences, tokens past the output, unreadable blocks
    and lengths past the bound: those rows stay as they were."""
    rng = np.random.default_rng(1)
    H, D = 2, 64
    cache = torch.from_numpy(_filled(rng, 8, 1, H, D, "bf16")).to(device)
    tables = torch.tensor([[3, 99], [1, -5], [6, 7]], dtype=torch.int32, device=device)
    lens = torch.tensor([20, 18, 1000], dtype=torch.int32, device=device)
    cu = torch.tensor([2, 30, 50, 70], dtype=torch.int32, device=device)
    k, v = kv4.gather_tokens_kv4(cache, tables, lens, 60, 32, cu_seqlens=cu)
    want_k, _ = k4.rows(cache[:, 0].cpu().numpy(), D)
    got = k[0].double().cpu().numpy()
    assert np.array_equal(got[2:18], want_k[3])     # 18..21: block 99
    assert np.array_equal(got[30:46], want_k[1])    # 46, 47: block -5
    assert np.array_equal(got[50:60], want_k[6][:10])  # cut by the output's end
    # the same with room: the third stops at the bound of 32
    out_k, _ = kv4.gather_tokens_kv4(cache, tables, lens, 100, 32, cu_seqlens=cu)
    assert np.array_equal(out_k[0, 66:82].double().cpu().numpy(), want_k[7])


def test_gather_batch_past_one_launch(device):
    rng = np.random.default_rng(2)
    lens = rng.integers(0, 20, size=1500)
    cache = _filled(rng, 64, 1, 1, 64, "fp16")
    tables = [[int(x) for x in rng.integers(0, 64, size=-(-n // 16))] for n in lens]
    k, v = kv4.gather_tokens_kv4(torch.from_numpy(cache).to(device),
                                 torch.from_numpy(ko.pad_block_tables(tables)).to(device),
                                 torch.from_numpy(lens.astype(np.int32)).to(device),
                                 int(lens.sum()), int(lens.max()), dtype=torch.float16)
    rk, rv = k4.rows(cache[:, 0], 64)
    for got, side in ((k, rk), (v, rv)):
        want = np.concatenate([side[t].reshape(-1, 1, 64)[:n] for t, n in zip(tables, lens) if n])
        assert np.array_equal(got[0].double().cpu().numpy(), want)


# ---------------------------------------------------------------------------
# decode attention
# ---------------------------------------------------------------------------
def _decode_setup(device, lens, Hq, Hkv, D, dtype, seed, spare=3):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens)
    n = int(sum(-(-int(x) // 16) for x in lens)) + spare
    cache = _filled(rng, n, 1, Hkv, D, dtype)[:, 0]
    tables = _tables(rng, lens, n)
    for t, x in zip(tables, lens):  # stale bytes behind the sequence's last token
        if x % 16:
            for side in (0, 1):
                for r in range(x % 16, 16):
                    cache[t[-1], :, side, 8 * D + r::16] = 255
                    for d in range(D):
                        cache[t[-1], :, side, k4.byte_of(side, D, r, d)[0]] = 0xC3
    q = random_bits(rng, (len(lens), Hq, D), dtype)
    return (rng, lens, tables, cache, q, torch.from_numpy(cache).to(device),
            to_device_bits(q, dtype, device),
            torch.from_numpy(ko.pad_block_tables(tables)).to(device),
            torch.from_numpy(lens.astype(np.int32)).to(device))


def _check_decode(out, q, cache, tables, lens, scale, D, dtype):
    k, v = k4.rows(cache, D)
    ref = ko.paged_decode_attention(ko.bits_to_float(q, dtype), np.nan_to_num(k), np.nan_to_num(v),
                                    ko.pad_block_tables(tables), lens, scale)
    got = out.double().cpu().numpy()
    err = np.linalg.norm(got - ref) / max(np.linalg.norm(ref), 1e-30)
    assert err <= 2e-3, err
    ulp = bf16_ulp(ref) if dtype == "bf16" else fp16_ulp(ref)
    bar = ulp + 1e-5 + 2.0 ** -17 * np.nanmax(np.abs(v))
    assert (np.abs(got - ref) <= bar).all(), np.abs(got - ref).max()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (8, 8, 128), (16, 1, 64), (6, 2, 256),
                                      (12, 6, 128), (9, 3, 64), (20, 20, 64), (7, 1, 128),
                                      (16, 1, 256)])
@pytest.mark.parametrize("nwg", [0, 1, 3, 1000])
def test_decode_matches_the_textbook(device, dtype, Hq, Hkv, D, nwg):
    lens = [1, 15, 16, 17, 31, 64, 65, 200, 517, 0, 1100, 127]
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, lens, Hq, Hkv, D, dtype,
                                                               Hq * 10 + D + nwg)
    out = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 1 / math.sqrt(D), 1100, n_workgroups=nwg)
    assert not out[9].any()
    _check_decode(out, q, cache, tables, lens, 1 / math.sqrt(D), D, dtype)


@pytest.mark.parametrize("lens", [[1], [16], [5000], [20000, 3], [700] * 40])
@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (4, 2, 64)])
def test_decode_lengths(device, lens, Hq, Hkv, D):
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, lens, Hq, Hkv, D, "bf16", 4)
    out = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 0.11, int(max(lens)))
    _check_decode(out, q, cache, tables, lens, 0.11, D, "bf16")


@pytest.mark.parametrize("scale", [0.0, -0.09, 3.0])
def test_decode_scales(device, scale):
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, [40, 333], 8, 2, 128,
                                                               "fp16", 6)
    out = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, scale, 333)
    _check_decode(out, q, cache, tables, lens, scale, 128, "fp16")


@pytest.mark.parametrize("batch", [5, 300])
@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (7, 1, 128), (6, 2, 256), (9, 3, 64)])
def test_planned_call_is_bit_identical(device, batch, Hq, Hkv, D):
    lens = np.random.default_rng(batch).integers(0, 260, size=batch)
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, lens, Hq, Hkv, D, "bf16", 9)
    longest = int(lens.max())
    plain = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 0.1, longest)
    plan = A.DecodePlan(bt, sl, longest, Hkv)
    for _ in range(2):
        planned = kv4.paged_decode_attention_kv4(dq, dc, None, None, 0.1, longest, plan=plan)
        assert torch.equal(plain.view(torch.int16), planned.view(torch.int16))


def test_decode_batch_above_one_launch(device):
    lens = np.random.default_rng(3).integers(0, 40, size=2500)
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, lens, 4, 2, 64, "bf16", 12)
    out = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 0.12, 40)
    _check_decode(out, q, cache, tables, lens, 0.12, 64, "bf16")


def test_decode_bound_strides_and_unreadable_blocks(device):
    """Lengths past the host bound, an output and a query inside wider
    buffers, a layer of a larger cache, block ids outside the pool (their tokens
    masked)."""
    Hq, Hkv, D = 8, 2, 128
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, [100, 90, 48], Hq, Hkv, D,
                                                               "bf16", 21)
    wide_cache = torch.full((dc.size(0), 3, Hkv, 2, 1088), 255, dtype=torch.uint8, device=device)
    wide_cache[:, 1] = dc
    wide_q = torch.zeros(3, Hq * D + 64, dtype=torch.bfloat16, device=device)
    wide_q[:, :Hq * D] = dq.flatten(1)
    wide_o = torch.full((3, Hq * D + 8), 5.0, dtype=torch.bfloat16, device=device)
    kv4.paged_decode_attention_kv4(wide_q[:, :Hq * D].unflatten(1, (Hq, D)), wide_cache[:, 1], bt,
                                   sl, 0.1, 64, out=wide_o[:, :Hq * D].unflatten(1, (Hq, D)))
    assert bool((wide_o[:, Hq * D:] == 5.0).all())
    _check_decode(wide_o[:, :Hq * D].unflatten(1, (Hq, D)), q, cache, tables, [64, 64, 48], 0.1, D,
                  "bf16")
    # the second block of sequence 0 unreadable, all of sequence 2
    bad = bt.clone()
    bad[0, 1] = dc.size(0)
    bad[2] = -1
    out = kv4.paged_decode_attention_kv4(dq, dc, bad, sl, 0.1, 100)
    k, v = (np.nan_to_num(x) for x in k4.rows(cache, D))
    keep = [i for i in range(100) if not 16 <= i < 32]
    kk = k[tables[0]].reshape(-1, Hkv, D)[keep]
    vv = v[tables[0]].reshape(-1, Hkv, D)[keep]
    fq = ko.bits_to_float(q, "bf16")
    for h in range(Hq):
        s = kk[:, h // 4] @ fq[0, h] * 0.1
        p = np.exp(s - s.max())
        want = p @ vv[:, h // 4] / p.sum()
        assert np.abs(out[0, h].double().cpu().numpy() - want).max() <= \
            2.0 ** -8 * np.abs(want).max() + 1e-5 + 2.0 ** -17 * np.abs(vv).max()
    assert not out[2].any()


def test_a_nan_group_shows_in_its_own_head_only(device):
    Hq, Hkv, D = 4, 2, 64
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, [50, 20], Hq, Hkv, D,
                                                               "bf16", 30)
    clean = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 0.1, 50)
    dc[tables[0][1], 1, 0, 8 * D] = 255  # K of kv head 1, token 16
    out = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 0.1, 50)
    assert torch.isnan(out[0, 2:].float()).all()
    assert torch.equal(out[0, :2], clean[0, :2]) and torch.equal(out[1], clean[1])


def test_a_larger_pool_past_32_bit_offsets(device):
    """Blocks whose byte offset passes 2^32."""
    Hq, Hkv, D = 4, 1, 128
    n, layers = 70000, 32  # 69632 bytes per block, 4.87e9 in all
    cache = torch.empty((n, layers, Hkv, 2, 1088), dtype=torch.uint8, device=device)
    rng = np.random.default_rng(2)
    lens = np.array([40, 16])
    tables = [[n - 1, 5, n - 70], [n - 3000]]
    x = random_bits(rng, (2, 56, Hkv, D), "bf16")
    slots = np.array([tables[0][i // 16] * 16 + i % 16 for i in range(40)]
                     + [tables[1][0] * 16 + i for i in range(16)])
    dx = to_device_bits(x, "bf16", device)
    kv4.reshape_and_cache_kv4(dx[0], dx[1], cache[:, 31], torch.from_numpy(slots).to(device))
    bt = torch.from_numpy(ko.pad_block_tables(tables)).to(device)
    sl = torch.from_numpy(lens.astype(np.int32)).to(device)
    gk, gv = kv4.gather_tokens_kv4(cache, bt, sl, 56, 40, layers=(31, 1))
    for side, got in ((0, gk), (1, gv)):
        f = ko.bits_to_float(x[side], "bf16")
        assert np.array_equal(got[0].double().cpu().numpy(), k4.decode(*k4.encode(f, "bf16")))
    q = random_bits(rng, (2, Hq, D), "bf16")
    out = kv4.paged_decode_attention_kv4(to_device_bits(q, "bf16", device), cache[:, 31], bt, sl,
                                         0.1, 40)
    small = _poisoned(4, 1, Hkv, D)
    f = ko.bits_to_float(x, "bf16")
    k4.append(f[0][None], f[1][None], small, np.concatenate([np.arange(40), np.arange(48, 64)]),
              "bf16")
    _check_decode(out, q, small[:, 0], [[0, 1, 2], [3]], lens, 0.1, D, "bf16")


def test_captured_calls_replay_and_share_nothing(device):
    """Two graphs captured on one stream, replayed on two at once, with eager
    calls and new inputs between: every replay equals the eager result."""
    Hq, Hkv, D = 28, 4, 128
    sets = [_decode_setup(device, [900, 3, 2500, 64], Hq, Hkv, D, "bf16", s) for s in (41, 42)]
    outs = [torch.empty_like(s[6]) for s in sets]
    graphs, side = [], torch.cuda.Stream()
    for s, o in zip(sets, outs):
        kv4.paged_decode_attention_kv4(s[6], s[5], s[7], s[8], 0.1, 2500)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            kv4.paged_decode_attention_kv4(s[6], s[5], s[7], s[8], 0.1, 2500, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        for s in sets:
            s[6].mul_(-1.25)
        want = [kv4.paged_decode_attention_kv4(s[6], s[5], s[7], s[8], 0.1, 2500) for s in sets]
        torch.cuda.synchronize()
        for _ in range(3):
            for st, g in zip(streams, graphs):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o.view(torch.int16), w.view(torch.int16))


def test_decode_on_another_stream_with_a_plan_of_the_first(device):
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, [300, 50], 28, 4, 128,
                                                               "bf16", 50)
    want = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 0.1, 300)
    plan = A.DecodePlan(bt, sl, 300, 4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = kv4.paged_decode_attention_kv4(dq, dc, None, None, 0.1, 300, plan=plan)
    st.synchronize()
    assert torch.equal(want, got)


def test_the_cache_through_the_block_ops(device):
    """A sequence's life: appended, swapped out to pinned memory and back into
    other blocks, compacted, read by both readers."""
    rng = np.random.default_rng(77)
    L, Hkv, D, n, B = 3, 2, 128, 32, 4
    lens = np.array([70, 33, 16, 5])
    cache = kv4.kv4_cache(n, L, Hkv, D, device)
    tables = _tables(rng, lens, n)
    slots = np.concatenate([[t[p // 16] * 16 + p % 16 for p in range(x)]
                            for t, x in zip(tables, lens)])
    x = random_bits(rng, (2, L, int(lens.sum()), Hkv, D), "bf16")
    dx = to_device_bits(x, "bf16", device)
    kv4.append_kv4(dx[0], dx[1], cache, torch.from_numpy(slots).to(device))
    q = to_device_bits(random_bits(rng, (B, 8, D), "bf16"), "bf16", device)
    sl = torch.from_numpy(lens.astype(np.int32)).to(device)

    def read(tables):
        bt = torch.from_numpy(ko.pad_block_tables(tables)).to(device)
        k, v = kv4.gather_tokens_kv4(cache, bt, sl, int(lens.sum()), int(lens.max()))
        outs = [kv4.paged_decode_attention_kv4(q, cache[:, l], bt, sl, 0.1, int(lens.max()))
                for l in range(L)]
        return [k, v] + outs

    before = read(tables)
    f = ko.bits_to_float(x, "bf16")
    for side in (0, 1):
        assert np.array_equal(before[side].double().cpu().numpy(),
                              k4.decode(*k4.encode(f[side], "bf16")))
    used = [b for t in tables for b in t]
    host = torch.empty((len(used), L, Hkv, 2, 1088), dtype=torch.uint8, pin_memory=True)
    ops.swap(used, list(range(len(used))), False, cache, host)
    torch.cuda.synchronize()
    cache.fill_(255)
    new = [int(b) for b in rng.permutation(n)[:len(used)]]
    ops.swap(list(range(len(used))), new, True, cache, host)
    moved = dict(zip(used, new))
    tables = [[moved[b] for b in t] for t in tables]
    after = read(tables)
    from aegaeon_amd.pool import plan_compaction, remap_tables
    src, dst = plan_compaction(new, range(n))
    if len(src):
        ops.defrag_blocks(cache, src, dst)
    compacted = read(remap_tables(tables, src, dst))
    for a, b, c in zip(before, after, compacted):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        assert torch.equal(a.view(torch.int16), c.view(torch.int16))


def test_refusals(device):
    cache = kv4.kv4_cache(4, 2, 4, 128, device)
    x = torch.zeros(2, 3, 4, 128, dtype=torch.bfloat16, device=device)
    slots = torch.zeros(3, dtype=torch.int64, device=device)
    with pytest.raises(ValueError, match="slot"):
        kv4.append_kv4(x, x, cache, slots[:2])
    with pytest.raises(ValueError, match="int64"):
        kv4.append_kv4(x, x, cache, slots.int())
    with pytest.raises(ValueError, match="dtype"):
        kv4.append_kv4(x.float(), x.float(), cache, slots)
    with pytest.raises(ValueError, match="dtype"):
        kv4.append_kv4(x, x.half(), cache, slots)
    with pytest.raises(ValueError, match="layers"):
        kv4.append_kv4(x[:1], x[:1], cache, slots)
    with pytest.raises(ValueError, match="uint8"):
        kv4.append_kv4(x, x, cache.view(torch.int8), slots)
    with pytest.raises(ValueError, match="R = "):
        kv4.append_kv4(x[..., :64].contiguous(), x[..., :64].contiguous(), cache, slots)
    with pytest.raises(ValueError, match="dense"):
        kv4.append_kv4(x[..., ::2], x[..., ::2], cache, slots)
    with pytest.raises(ValueError, match="densely"):
        kv4.append_kv4(x[:, :, :2], x[:, :, :2], cache[:, :, ::2], slots)
    bt = torch.zeros(1, 2, dtype=torch.int32, device=device)
    sl = torch.ones(1, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="dtype"):
        kv4.gather_tokens_kv4(cache, bt, sl, 1, 1, dtype=torch.float32)
    with pytest.raises(ValueError, match="layer range"):
        kv4.gather_tokens_kv4(cache, bt, sl, 1, 1, layers=(1, 2))
    with pytest.raises(AegkvError):
        kv4.gather_tokens_kv4(cache, bt, sl, 1, 100)
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="kv_cache"):
        kv4.paged_decode_attention_kv4(q, cache, bt, sl, 0.1, 16)
    with pytest.raises(ValueError, match="workspace"):
        kv4.paged_decode_attention_kv4(q, cache[:, 0], bt, sl, 0.1, 16,
                                       workspace=torch.empty(16, dtype=torch.uint8, device=device))
    plan = A.DecodePlan(bt, sl, 16, 4)
    with pytest.raises(ValueError, match="plan"):
        kv4.paged_decode_attention_kv4(q, cache[:, 0], None, None, 0.1, 32, plan=plan)
    with pytest.raises(ValueError, match="required"):
        kv4.paged_decode_attention_kv4(q, cache[:, 0], None, None, 0.1, 16)
    with pytest.raises(AegkvError):
        kv4.paged_decode_attention_kv4(torch.zeros(1, 6, 128, dtype=torch.bfloat16, device=device),
                                       cache[:, 0], bt, sl, 0.1, 16)  # 6 heads over 4

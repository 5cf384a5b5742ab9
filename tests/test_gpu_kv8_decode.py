"""GPU parity of decode attention over the 8-bit KV cache with the oracle's
float64 textbook over the stored values.

The stored values are exact in 16 bits and the arithmetic past them is the 16-bit
cache's, so its bars are test_gpu_attention.py's: 2e-3 relative L2, and per
element one ulp of the output type plus 1e-5 and 2^-17 of the largest |v| (each
softmax weight keeps 16 significant bits)."""
import math

import numpy as np
import pytest
import torch

from aegaeon_amd import attention as A
from aegaeon_amd import kv8, rotary
from aegaeon_amd._lib import AegkvError
from oracle import kv8_oracle as k8
from oracle import kv_oracle as ko
from tests.kvtest_utils import bf16_ulp, fp16_ulp, random_bits, to_device_bits
from tests.test_gpu_kv8 import _filled, _rows, _slots, _tables

pytestmark = pytest.mark.gpu


def poison_behind(cache, tables, lens, heads, dim):
    """NaN codes behind each sequence's last token, as another sequence may have
    left them."""
    for t, n in zip(tables, lens):
        for r in range(n % 16, 16) if n % 16 else ():
            for side in (0, 1):
                for h in range(heads):
                    at = [(2 * h + side) * 16 * dim + k8.byte_of(side, dim, r, d)
                          for d in range(dim)]
                    cache[t[-1], at] = 0xFF if r & 1 else 0x7F


def _setup(device, lens, Hq, Hkv, D, dtype, seed, spare=3):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens)
    n = int(sum(-(-int(x) // 16) for x in lens)) + spare
    cache = _filled(rng, n, 1, Hkv, D, dtype)[:, 0]
    tables = _tables(rng, lens, n)
    poison_behind(cache, tables, lens, Hkv, D)
    q = random_bits(rng, (len(lens), Hq, D), dtype)
    return (rng, lens, tables, cache, q, torch.from_numpy(cache).to(device),
            to_device_bits(q, dtype, device),
            torch.from_numpy(ko.pad_block_tables(tables)).to(device),
            torch.from_numpy(lens.astype(np.int32)).to(device))


def _check(out, q, cache, tables, lens, scale, Hkv, D, dtype):
    k, v = (np.nan_to_num(x) for x in k8.rows(cache, Hkv, D))
    ref = ko.paged_decode_attention(ko.bits_to_float(q, dtype), k, v, ko.pad_block_tables(tables),
                                    lens, scale)
    got = out.double().cpu().numpy()
    err = np.linalg.norm(got - ref) / max(np.linalg.norm(ref), 1e-30)
    assert err <= 2e-3, err
    ulp = bf16_ulp(ref) if dtype == "bf16" else fp16_ulp(ref)
    bar = ulp + 1e-5 + 2.0 ** -17 * np.abs(v).max()
    assert (np.abs(got - ref) <= bar).all(), np.abs(got - ref).max()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (8, 8, 128), (16, 1, 64), (6, 2, 256),
                                      (12, 6, 128), (9, 3, 64), (20, 20, 64), (7, 1, 128),
                                      (16, 1, 256), (40, 4, 128)])
@pytest.mark.parametrize("nwg", [0, 1, 3, 1000])
def test_decode_matches_the_textbook(device, dtype, Hq, Hkv, D, nwg):
    lens = [1, 15, 16, 17, 31, 64, 65, 200, 517, 0, 1100, 127]
    rng, lens, tables, cache, q, dc, dq, bt, sl = _setup(device, lens, Hq, Hkv, D, dtype,
                                                        Hq * 10 + D + nwg)
    out = kv8.paged_decode_attention_kv8(dq, dc, bt, sl, 1 / math.sqrt(D), 1100, n_workgroups=nwg)
    assert not out[9].any()
    _check(out, q, cache, tables, lens, 1 / math.sqrt(D), Hkv, D, dtype)


@pytest.mark.parametrize("lens", [[1], [16], [5000], [20000, 3], [700] * 40])
@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (4, 2, 64)])
def test_decode_lengths(device, lens, Hq, Hkv, D):
    rng, lens, tables, cache, q, dc, dq, bt, sl = _setup(device, lens, Hq, Hkv, D, "bf16", 4)
    out = kv8.paged_decode_attention_kv8(dq, dc, bt, sl, 0.11, int(max(lens)))
    _check(out, q, cache, tables, lens, 0.11, Hkv, D, "bf16")


@pytest.mark.parametrize("scale", [0.0, -0.09, 3.0])
def test_decode_scales(device, scale):
    rng, lens, tables, cache, q, dc, dq, bt, sl = _setup(device, [40, 333], 8, 2, 128, "fp16", 6)
    out = kv8.paged_decode_attention_kv8(dq, dc, bt, sl, scale, 333)
    _check(out, q, cache, tables, lens, scale, 2, 128, "fp16")


@pytest.mark.parametrize("batch", [5, 300])
@pytest.mark.parametrize("Hq,Hkv,D", [(28, 4, 128), (7, 1, 128), (6, 2, 256), (9, 3, 64)])
def test_planned_call_is_bit_identical(device, batch, Hq, Hkv, D):
    lens = np.random.default_rng(batch).integers(0, 260, size=batch)
    rng, lens, tables, cache, q, dc, dq, bt, sl = _setup(device, lens, Hq, Hkv, D, "bf16", 9)
    longest = int(lens.max())
    plain = kv8.paged_decode_attention_kv8(dq, dc, bt, sl, 0.1, longest)
    plan = A.DecodePlan(bt, sl, longest, Hkv)
    for _ in range(2):
        planned = kv8.paged_decode_attention_kv8(dq, dc, None, None, 0.1, longest, plan=plan)
        assert torch.equal(plain.view(torch.int16), planned.view(torch.int16))


def test_decode_batch_above_one_launch(device):
    lens = np.random.default_rng(3).integers(0, 40, size=2500)
    rng, lens, tables, cache, q, dc, dq, bt, sl = _setup(device, lens, 4, 2, 64, "bf16", 12)
    out = kv8.paged_decode_attention_kv8(dq, dc, bt, sl, 0.12, 40)
    _check(out, q, cache, tables, lens, 0.12, 2, 64, "bf16")


def test_decode_bound_strides_and_unreadable_blocks(device):
    """Lengths past the host bound, an output and a query inside wider buffers, a
    layer of a larger cache, block ids outside the pool (their tokens masked)."""
    Hq, Hkv, D = 8, 2, 128
    R = k8.block_bytes(Hkv, D)
    rng, lens, tables, cache, q, dc, dq, bt, sl = _setup(device, [100, 90, 48], Hq, Hkv, D, "bf16",
                                                        21)
    wide_cache = torch.full((dc.size(0), 3, R), 255, dtype=torch.uint8, device=device)
    wide_cache[:, 1] = dc
    wide_q = torch.zeros(3, Hq * D + 64, dtype=torch.bfloat16, device=device)
    wide_q[:, :Hq * D] = dq.flatten(1)
    wide_o = torch.full((3, Hq * D + 8), 5.0, dtype=torch.bfloat16, device=device)
    out = wide_o[:, :Hq * D].unflatten(1, (Hq, D))
    kv8.paged_decode_attention_kv8(wide_q[:, :Hq * D].unflatten(1, (Hq, D)), wide_cache[:, 1], bt,
                                   sl, 0.1, 64, out=out)
    assert bool((wide_o[:, Hq * D:] == 5.0).all())
    _check(out, q, cache, tables, [64, 64, 48], 0.1, Hkv, D, "bf16")
    # the second block of sequence 0 unreadable, all of sequence 2
    bad = bt.clone()
    bad[0, 1] = dc.size(0)
    bad[2] = -1
    out = kv8.paged_decode_attention_kv8(dq, dc, bad, sl, 0.1, 100)
    k, v = (np.nan_to_num(x) for x in k8.rows(cache, Hkv, D))
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


@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (32, 2)])
def test_a_nan_shows_in_its_own_head_and_dim_only(device, Hq, Hkv):
    """A NaN key: its kv head's queries of that sequence; a NaN value: that dim
    of theirs."""
    D, G = 64, Hq // Hkv
    rng, lens, tables, cache, q, dc, dq, bt, sl = _setup(device, [50, 20], Hq, Hkv, D, "bf16", 30)
    clean = kv8.paged_decode_attention_kv8(dq, dc, bt, sl, 0.1, 50)
    blk, held = tables[0][1], dc.clone()
    dc[blk, 2 * 16 * D + k8.byte_of(0, D, 3, 7)] = 0xFF  # K of kv head 1, token 19
    out = kv8.paged_decode_attention_kv8(dq, dc, bt, sl, 0.1, 50)
    assert torch.isnan(out[0, G:].float()).all()
    assert torch.equal(out[0, :G], clean[0, :G]) and torch.equal(out[1], clean[1])
    dc.copy_(held)
    dc[blk, 3 * 16 * D + k8.byte_of(1, D, 3, 7)] = 0x7F
    out = kv8.paged_decode_attention_kv8(dq, dc, bt, sl, 0.1, 50)
    assert torch.isnan(out[0, G:, 7].float()).all()
    out[0, G:, 7] = clean[0, G:, 7]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_small_weights_are_kept(device, dtype):
    """Thousands of keys of 2^-24 of the largest weight beside one key: together
    they are not nothing."""
    n, D = 4096, 64
    R = k8.block_bytes(1, D)
    cache = np.zeros((n // 16, 1, R), dtype=np.uint8)
    k = np.zeros((1, n, 1, D))
    k[0, 0, 0, 0] = 24.0
    v = np.ones((1, n, 1, D))
    v[0, 0] = 0.0
    k8.append(k, v, cache, np.arange(n), dtype)
    q = np.zeros((1, 1, D))
    q[..., 0] = 1.0
    dq = to_device_bits(ko.float_to_bits(q, dtype), dtype, device)
    out = kv8.paged_decode_attention_kv8(
        dq, torch.from_numpy(cache[:, 0]).to(device),
        torch.arange(n // 16, dtype=torch.int32, device=device)[None],
        torch.tensor([n], dtype=torch.int32, device=device), math.log(2.0), n)
    want = 4095 * 2.0 ** -24 / (1 + 4095 * 2.0 ** -24)
    # P in two 16-bit parts (bf16: 16 bits of each weight), the output's rounding
    assert abs(float(out[0, 0, 5]) / want - 1) < 2.0 ** -8 + 2.0 ** -12


def test_captured_calls_replay_and_share_nothing(device):
    """Two graphs captured on one stream, replayed on two at once, with eager
    calls and new inputs between: every replay equals the eager result."""
    Hq, Hkv, D = 28, 4, 128
    sets = [_setup(device, [900, 3, 2500, 64], Hq, Hkv, D, "bf16", s) for s in (41, 42)]
    outs = [torch.empty_like(s[6]) for s in sets]
    graphs, side = [], torch.cuda.Stream()
    for s, o in zip(sets, outs):
        kv8.paged_decode_attention_kv8(s[6], s[5], s[7], s[8], 0.1, 2500)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            kv8.paged_decode_attention_kv8(s[6], s[5], s[7], s[8], 0.1, 2500, out=o)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        for s in sets:
            s[6].mul_(-1.25)
        want = [kv8.paged_decode_attention_kv8(s[6], s[5], s[7], s[8], 0.1, 2500) for s in sets]
        torch.cuda.synchronize()
        for _ in range(3):
            for st, g in zip(streams, graphs):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o.view(torch.int16), w.view(torch.int16))


def test_decode_on_another_stream_with_a_plan_of_the_first(device):
    rng, lens, tables, cache, q, dc, dq, bt, sl = _setup(device, [300, 50], 28, 4, 128, "bf16", 50)
    want = kv8.paged_decode_attention_kv8(dq, dc, bt, sl, 0.1, 300)
    plan = A.DecodePlan(bt, sl, 300, 4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = kv8.paged_decode_attention_kv8(dq, dc, None, None, 0.1, 300, plan=plan)
    st.synchronize()
    assert torch.equal(want, got)


def test_a_larger_pool_past_32_bit_offsets(device):
    H, D, n, layers = 1, 128, 40000, 32  # 135168 bytes per block, 5.4e9 in all
    cache = torch.empty((n, layers, k8.block_bytes(H, D)), dtype=torch.uint8, device=device)
    rng = np.random.default_rng(2)
    tables, lens = [[n - 1, 5, n - 70], [n - 3000]], np.array([40, 16])
    x = _rows(rng, (2, 56, H, D), "bf16")
    dx = to_device_bits(x, "bf16", device)
    kv8.reshape_and_cache_kv8(dx[0], dx[1], cache[:, 31], torch.from_numpy(
        _slots(tables, [(0, 40), (0, 16)])).to(device))
    q = random_bits(rng, (2, 4, D), "bf16")
    out = kv8.paged_decode_attention_kv8(
        to_device_bits(q, "bf16", device), cache[:, 31],
        torch.from_numpy(ko.pad_block_tables(tables)).to(device),
        torch.from_numpy(lens.astype(np.int32)).to(device), 0.1, 40)
    small = np.zeros((4, 1, k8.block_bytes(H, D)), dtype=np.uint8)
    f = ko.bits_to_float(x, "bf16")
    k8.append(f[0][None], f[1][None], small, np.concatenate([np.arange(40), 48 + np.arange(16)]),
              "bf16")
    _check(out, q, small[:, 0], [[0, 1, 2], [3]], lens, 0.1, H, D, "bf16")


def test_a_decode_loop_of_turned_appends_and_attention(device):
    """Prompts turned and appended, then steps of one token each: turn, append,
    attend, over two layers that share a plan per step."""
    rng = np.random.default_rng(8)
    Hq, Hkv, D, L = 14, 2, 128, 2
    lens = np.array([30, 1, 47])
    tables = _tables(rng, lens + 20, 12)
    table = rotary.rotary_table(100, D, device=device)
    t = table.cpu().numpy()
    cache = np.zeros((12, L, k8.block_bytes(Hkv, D)), dtype=np.uint8)
    dev = kv8.kv8_cache(12, L, Hkv, D, device)
    bt = torch.from_numpy(ko.pad_block_tables(tables)).to(device)

    def turn(layer, spans):
        slots = _slots(tables, spans)
        pos = np.array([p for a, b in spans for p in range(a, b)])
        q, k, v = (_rows(rng, (len(pos), h, D), "bf16") for h in (Hq, Hkv, Hkv))
        out = kv8.rotary_and_cache_kv8(*(to_device_bits(x, "bf16", device) for x in (q, k, v)),
                                       dev[:, layer], torch.from_numpy(slots).to(device),
                                       torch.from_numpy(pos).to(device), table)
        fq, fk, fv = (ko.bits_to_float(x, "bf16") for x in (q, k, v))
        k8.append(k8.turned(fk, pos, t, False)[None], fv[None], cache[:, layer:layer + 1], slots,
                  "bf16")
        return out, ko.float_to_bits(k8.turned(fq, pos, t, False).astype(np.float64), "bf16")

    for layer in range(L):
        turn(layer, [(0, int(n)) for n in lens])
    for step in range(5):
        lens = lens + 1
        sl = torch.from_numpy(lens.astype(np.int32)).to(device)
        plan = A.DecodePlan(bt, sl, int(lens.max()), Hkv)
        for layer in range(L):
            q, want_q = turn(layer, [(int(n) - 1, int(n)) for n in lens])
            out = kv8.paged_decode_attention_kv8(q, dev[:, layer], None, None, 0.09,
                                                 int(lens.max()), plan=plan)
            assert np.array_equal(dev[:, layer].cpu().numpy(), cache[:, layer])
            _check(out, want_q, cache[:, layer], tables, lens, 0.09, Hkv, D, "bf16")


@pytest.mark.parametrize("planned", [False, True])
def test_a_captured_step_equals_the_eager_one(device, planned):
    """A step's append with rotation and its attention in one graph, replayed over
    steps that cross block edges, a padded row among them: cache and outputs are
    those of the eager calls, bit for bit."""
    rng = np.random.default_rng(15)
    Hq, Hkv, D, bound = 28, 4, 128, 64
    lens = np.array([13, 30, 1, 0])
    tables = _tables(rng, lens + 20, 12)
    bt = torch.from_numpy(ko.pad_block_tables(tables)).to(device)
    start = torch.from_numpy(_filled(rng, 12, 1, Hkv, D, "bf16")[:, 0]).to(device)
    table = rotary.rotary_table(100, D, device=device)
    T = len(lens)
    q, k, v = (torch.zeros(T, h, D, dtype=torch.bfloat16, device=device) for h in (Hq, Hkv, Hkv))
    slots, pos = (torch.zeros(T, dtype=torch.int64, device=device) for _ in range(2))
    sl = torch.ones(T, dtype=torch.int32, device=device)

    def step(cache):
        turned = kv8.rotary_and_cache_kv8(q, k, v, cache, slots, pos, table)
        plan = A.DecodePlan(bt, sl, bound, Hkv) if planned else None
        return kv8.paged_decode_attention_kv8(turned, cache, bt, sl, 0.09, bound, plan=plan)

    eager, captured = start.clone(), start.clone()
    step(captured)  # what a first call sets up
    captured.copy_(start)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(captured)
    for _ in range(6):
        active = lens > 0
        lens = lens + active
        for dst, h in ((q, Hq), (k, Hkv), (v, Hkv)):
            dst.copy_(to_device_bits(_rows(rng, (T, h, D), "bf16"), "bf16", device))
        slots.copy_(torch.tensor([t[(n - 1) // 16] * 16 + (n - 1) % 16 if n else -1
                                  for t, n in zip(tables, lens.tolist())]))
        pos.copy_(torch.from_numpy(np.maximum(lens - 1, 0)))
        sl.copy_(torch.from_numpy(lens.astype(np.int32)))
        want = step(eager)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, eager)
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))
        assert not out[3].any()


def test_refusals(device):
    cache = kv8.kv8_cache(4, 2, 4, 128, device)
    bt = torch.zeros(1, 2, dtype=torch.int32, device=device)
    sl = torch.ones(1, dtype=torch.int32, device=device)
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="kv_cache"):
        kv8.paged_decode_attention_kv8(q, cache, bt, sl, 0.1, 16)
    with pytest.raises(ValueError, match="R = "):
        kv8.paged_decode_attention_kv8(q, cache[:, 0, :-16], bt, sl, 0.1, 16)
    with pytest.raises(ValueError, match="dense"):
        kv8.paged_decode_attention_kv8(q, kv8.kv8_cache(4, 1, 4, 128, device).view(4, -1)
                                       .t().contiguous().t(), bt, sl, 0.1, 16)
    with pytest.raises(ValueError, match="workspace"):
        kv8.paged_decode_attention_kv8(q, cache[:, 0], bt, sl, 0.1, 16,
                                       workspace=torch.empty(16, dtype=torch.uint8, device=device))
    plan = A.DecodePlan(bt, sl, 16, 4)
    with pytest.raises(ValueError, match="plan"):
        kv8.paged_decode_attention_kv8(q, cache[:, 0], None, None, 0.1, 32, plan=plan)
    with pytest.raises(ValueError, match="required"):
        kv8.paged_decode_attention_kv8(q, cache[:, 0], None, None, 0.1, 16)
    for bad in (float("inf"), float("nan")):
        with pytest.raises(AegkvError):
            kv8.paged_decode_attention_kv8(q, cache[:, 0], bt, sl, bad, 16)
    with pytest.raises(AegkvError):
        kv8.paged_decode_attention_kv8(torch.zeros(1, 6, 128, dtype=torch.bfloat16, device=device),
                                       cache[:, 0], bt, sl, 0.1, 16)  # 6 heads over 4

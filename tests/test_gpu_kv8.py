"""GPU parity of the 8-bit KV cache's writes and de-page, and of the rotating
appends into either cache, with the oracle: every byte of the cache and every
16-bit value exactly (the rotation's operations are rounded one by one on both
sides, so its results too)."""
import threading

import numpy as np
import pytest
import torch

from aegaeon_amd import attention as A
from aegaeon_amd import kv8, ops, rotary
from aegaeon_amd._lib import AegkvError
from oracle import kv8_oracle as k8
from oracle import kv_oracle as ko
from tests.kvtest_utils import random_bits, to_bits, to_device_bits

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _poisoned(n, layers, heads, dim):
    return np.full((n, layers, k8.block_bytes(heads, dim)), 0xFF, dtype=np.uint8)


def _rows(rng, shape, dtype):
    """Rows whose channels and tokens differ much in size, as bits."""
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[-1])) \
        * np.exp(rng.standard_normal(shape[:-1]))[..., None]
    return ko.float_to_bits(x, dtype)


def _append(device, key, value, cache, slots, dtype, dev=None):
    """Both sides append the same rows (uint16 bits [L, T, Hkv, D])."""
    dev = torch.from_numpy(cache).to(device) if dev is None else dev
    slots = np.asarray(slots, dtype=np.int64)
    kv8.append_kv8(to_device_bits(key, dtype, device), to_device_bits(value, dtype, device), dev,
                   torch.from_numpy(slots).to(device))
    k8.append(ko.bits_to_float(key, dtype), ko.bits_to_float(value, dtype), cache, slots, dtype)
    return dev


def _slots(tables, spans):
    """Slots of positions [a, b) of each sequence."""
    return np.array([t[p // 16] * 16 + p % 16 for t, (a, b) in zip(tables, spans)
                     for p in range(a, b)], dtype=np.int64)


def _tables(rng, lens, pool):
    ids = [int(x) for x in rng.permutation(pool)]
    return [[ids.pop() for _ in range(-(-int(x) // 16))] for x in lens]


def _filled(rng, n, layers, heads, dim, dtype):
    """A cache whose every slot was written, as the oracle holds it."""
    cache = _poisoned(n, layers, heads, dim)
    x = ko.bits_to_float(_rows(rng, (2, layers, n * 16, heads, dim), dtype), dtype)
    k8.append(x[0], x[1], cache, np.arange(n * 16), dtype)
    return cache


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("L,H,D", [(1, 1, 64), (3, 4, 128), (2, 3, 256), (2, 5, 64)])
def test_prompts_then_steps(device, dtype, L, H, D):
    """Prompts of uneven lengths, then single tokens whose sizes grow and shrink,
    then drafted ones: the whole cache equals the oracle's after each call,
    untouched bytes included."""
    rng = np.random.default_rng(L * 100 + H * 10 + D)
    lens = [1, 37, 16, 15, 33, 2]
    tables = _tables(rng, [x + 24 for x in lens], 30)
    cache, dev = _poisoned(30, L, H, D), None
    at = list(lens)
    spans = [(0, x) for x in lens]
    for step in range(14):
        slots = _slots(tables, spans)
        if step == 3:  # padding before, between and behind
            slots = np.concatenate([[-1], slots[:2], [30 * 16, -7], slots[2:], [-1]])
        gain = 2.0 ** rng.integers(-6, 7)
        k, v = (ko.float_to_bits(ko.bits_to_float(_rows(rng, (L, len(slots), H, D), dtype), dtype)
                                 * gain, dtype) for _ in range(2))
        dev = _append(device, k, v, cache, slots, dtype, dev)
        assert np.array_equal(dev.cpu().numpy(), cache), step
        new = [3 if step == 9 else 1] * len(lens)
        spans = [(a, a + m) for a, m in zip(at, new)]
        at = [a + m for a, m in zip(at, new)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("order", ["sorted", "mixed"])
def test_append_of_every_16_bit_pattern(device, dtype, D, order):
    """All 65536 patterns: zeros, subnormals, infinities and NaN among them, in
    blocks of like magnitude and of any."""
    bits = np.arange(1 << 16, dtype=np.uint16)
    if order == "mixed":
        bits = np.random.default_rng(5).permutation(bits)
    T = (1 << 16) // D
    k = bits.reshape(1, T, 1, D).copy()
    v = k[:, ::-1].copy()
    cache = _poisoned(T // 16 + 1, 1, 1, D)
    with np.errstate(over="ignore", invalid="ignore"):
        dev = _append(device, k, v, cache, np.arange(T) + 3, dtype)
    assert np.array_equal(dev.cpu().numpy(), cache)


@pytest.mark.parametrize("slots", [
    [20, 19, 18, 17], [31, 16, 20], [16, 16, 17], [21, 20, 20, 22, 20], [40, 21, 22, 63, 5, 0]])
def test_slots_in_any_order_within_a_block(device, slots):
    """Descending, scattered, the same slot twice (the later row counts), the tokens
    of a block next to each other."""
    rng = np.random.default_rng(len(slots) + slots[0])
    cache = _filled(rng, 4, 2, 3, 128, "bf16")
    k, v = (_rows(rng, (2, len(slots), 3, 128), "bf16") for _ in range(2))
    dev = _append(device, k, v, cache, slots, "bf16")
    assert np.array_equal(dev.cpu().numpy(), cache)


@pytest.mark.parametrize("n", [46, 47, 48, 64, 200])
@pytest.mark.parametrize("before", [0, 5])
def test_places_given_many_times(device, n, before):
    """The last row for each place counts, however many there are for one block: a
    batch padded with rows for one slot."""
    rng = np.random.default_rng(n + before)
    cache = _filled(rng, 4, 2, 3, 128, "bf16")
    slots = [0] * before + [int(x) for x in 16 + rng.integers(0, 16, n)] + [32] * n
    k, v = (_rows(rng, (2, len(slots), 3, 128), "bf16") for _ in range(2))
    dev = _append(device, k, v, cache, slots, "bf16")
    assert np.array_equal(dev.cpu().numpy(), cache)


@pytest.mark.parametrize("tokens,layers", [(700, 28), (1500, 8), (4100, 1), (4096, 4)])
def test_many_tokens(device, tokens, layers):
    """Counts past which a wave takes several tokens' runs, single tokens and
    prompts mixed."""
    rng = np.random.default_rng(tokens)
    H, D = 4, 64
    lens = []
    while sum(lens) < tokens:
        lens.append(int(rng.choice([1, 1, 1, 1, 2, 5, 16, 17, 40])))
    pool = sum(-(-(x + 15) // 16) for x in lens)
    starts = rng.integers(0, 16, size=len(lens))
    tables = _tables(rng, [x + s for x, s in zip(lens, starts)], pool)
    slots = _slots(tables, [(int(s), int(s) + x) for x, s in zip(lens, starts)])
    k, v = (_rows(rng, (1, len(slots), H, D), "bf16").repeat(layers, 0) for _ in range(2))
    cache = np.zeros((pool, 1, k8.block_bytes(H, D)), dtype=np.uint8)
    dev = torch.zeros((pool, layers, cache.shape[2]), dtype=torch.uint8, device=device)
    dk, dv = to_device_bits(k, "bf16", device), to_device_bits(v, "bf16", device)
    kv8.append_kv8(dk, dv, dev, torch.from_numpy(slots).to(device))
    k8.append(ko.bits_to_float(k[:1], "bf16"), ko.bits_to_float(v[:1], "bf16"), cache, slots,
              "bf16")
    want = torch.from_numpy(cache).to(device)
    assert bool((dev == want).all())


def test_append_strided_rows_and_layer_view(device):
    """Rows that are slices of a fused projection, one layer of a cache of
    several: the other layers' bytes stay."""
    rng = np.random.default_rng(8)
    T, H, D = 37, 4, 128
    fused = _rows(rng, (T, 12 * D), "bf16")
    dev_fused = to_device_bits(fused, "bf16", device)
    key = dev_fused[:, 4 * D:8 * D].unflatten(1, (H, D))
    value = dev_fused[:, 8 * D:].unflatten(1, (H, D))
    cache = _poisoned(6, 3, H, D)
    dev = torch.from_numpy(cache).to(device)
    slots = np.arange(T) + 20
    kv8.reshape_and_cache_kv8(key, value, dev[:, 1], torch.from_numpy(slots).to(device))
    f = ko.bits_to_float(fused, "bf16")
    k8.append(f[None, :, 4 * D:8 * D].reshape(1, T, H, D), f[None, :, 8 * D:].reshape(1, T, H, D),
              cache[:, 1:2], slots, "bf16")
    assert np.array_equal(dev.cpu().numpy(), cache)


def test_append_of_nothing(device):
    cache = kv8.kv8_cache(2, 1, 2, 64, device).fill_(7)
    x = torch.empty(1, 0, 2, 64, dtype=torch.float16, device=device)
    none = torch.empty(0, dtype=torch.int64, device=device)
    kv8.append_kv8(x, x, cache, none)
    table = rotary.rotary_table(4, 64, device=device)
    q = kv8.rotary_and_cache_kv8(x[0], x[0], x[0], cache[:, 0], none, none, table)
    assert q.shape == (0, 2, 64)
    kc = torch.zeros(2, 16, 2, 64, dtype=torch.float16, device=device)
    rotary.rotary_and_cache(x[0], x[0], x[0], kc, kc.clone(), none, none, table)
    one = torch.ones(1, 2, 64, dtype=torch.float16, device=device)
    kv8.reshape_and_cache_kv8(one, one, cache[:, 0], torch.tensor([-1], device=device))
    assert bool((cache == 7).all())


# ---------------------------------------------------------------------------
# the rotating appends
# ---------------------------------------------------------------------------
def _turn_setup(device, T, Hq, Hkv, D, rot, dtype, seed, max_pos=500):
    rng = np.random.default_rng(seed)
    fused = _rows(rng, (T, (Hq + 2 * Hkv) * D + 16), dtype)
    dev = to_device_bits(fused, dtype, device)
    sizes = [Hq * D, Hkv * D, Hkv * D]
    q, k, v = (x.unflatten(1, (-1, D)) for x in dev[:, :sum(sizes)].split(sizes, 1))
    f = ko.bits_to_float(fused, dtype)
    fq, fk, fv = (x.reshape(T, -1, D) for x in np.split(f[:, :sum(sizes)], np.cumsum(sizes)[:-1], 1))
    table = rotary.rotary_table(max_pos, rot, device=device)
    return rng, (q, k, v), (fq, fk, fv), table, table.cpu().numpy()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,D,rot", [(28, 4, 128, 128), (2, 2, 64, 32), (6, 2, 256, 256),
                                          (9, 3, 80, 80), (5, 1, 96, 48), (40, 40, 128, 16),
                                          (1, 1, 512, 512)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T", [1, 45])
def test_rotary_append_to_the_16_bit_cache(device, dtype, Hq, Hkv, D, rot, interleaved, T):
    rng, (q, k, v), (fq, fk, fv), table, t = _turn_setup(device, T, Hq, Hkv, D, rot, dtype,
                                                        Hq + D + rot + T)
    positions = rng.integers(0, 500, size=T)
    slots = rng.permutation(6 * 16)[:T].astype(np.int64)
    if T > 3:
        slots[1], slots[7] = -1, 6 * 16
    cache = torch.full((6, 2, 2, 16, Hkv, D), 7.0, dtype=DTYPES[dtype], device=device)
    out_key = torch.empty_like(k, memory_format=torch.contiguous_format)
    out = rotary.rotary_and_cache(q, k, v, cache[:, 1, 0], cache[:, 1, 1],
                                  torch.from_numpy(slots).to(device),
                                  torch.from_numpy(positions).to(device), table,
                                  interleaved=interleaved, out_key=out_key)
    want_q = ko.float_to_bits(k8.turned(fq, positions, t, interleaved).astype(np.float64), dtype)
    want_k = ko.float_to_bits(k8.turned(fk, positions, t, interleaved).astype(np.float64), dtype)
    assert np.array_equal(to_bits(out), want_q)
    assert np.array_equal(to_bits(out_key), want_k)
    want = np.full((6, 2, 2, 16, Hkv, D), ko.float_to_bits(np.array(7.0), dtype))
    for i, s in enumerate(slots):
        if 0 <= s < 6 * 16:
            want[s // 16, 1, 0, s % 16] = want_k[i]
            want[s // 16, 1, 1, s % 16] = ko.float_to_bits(fv[i], dtype)
    assert np.array_equal(to_bits(cache), want)


def test_rotary_append_equals_rotation_then_append(device):
    """In place on the rows of a fused projection, and as two steps: the caches
    are the same bit for bit; another block size."""
    rng, (q, k, v), _, table, _ = _turn_setup(device, 33, 28, 4, 128, 64, "bf16", 3)
    slots = torch.from_numpy(rng.permutation(3 * 32)[:33].astype(np.int64)).to(device)
    positions = torch.arange(33, device=device) + 100
    caches = [torch.zeros(3, 2, 32, 4, 128, dtype=torch.bfloat16, device=device) for _ in range(2)]
    key = torch.empty(k.shape, dtype=k.dtype, device=device)
    out = rotary.rotary_and_cache(q, k, v, caches[0][:, 0], caches[0][:, 1], slots, positions,
                                  table, out_key=key)
    A.reshape_and_cache_flash(key, v, caches[1][:, 0], caches[1][:, 1], slots)
    assert torch.equal(caches[0].view(torch.int16), caches[1].view(torch.int16))
    caches[0].zero_()
    back = rotary.rotary_and_cache(q, k, v, caches[0][:, 0], caches[0][:, 1], slots, positions,
                                   table, out=q, out_key=k)
    assert back is q and torch.equal(q, out) and torch.equal(k, key)
    assert torch.equal(caches[0].view(torch.int16), caches[1].view(torch.int16))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,D,rot", [(28, 4, 128, 128), (2, 2, 64, 32), (6, 2, 256, 256),
                                          (7, 1, 256, 32), (40, 40, 128, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_append_to_the_8_bit_cache(device, dtype, Hq, Hkv, D, rot, interleaved):
    """A prompt's tokens, then single ones that join their blocks."""
    lens = [40, 1, 16, 21]
    rng, (q, k, v), (fq, fk, fv), table, t = _turn_setup(device, sum(lens) + 4, Hq, Hkv, D, rot,
                                                        dtype, Hq + D + rot)
    tables = _tables(rng, [x + 1 for x in lens], 9)
    cache = _poisoned(9, 2, Hkv, D)
    dev = torch.from_numpy(cache).to(device)
    n = sum(lens)
    for rows, spans in ((slice(0, n), [(0, x) for x in lens]),
                        (slice(n, n + 4), [(x, x + 1) for x in lens])):
        slots = _slots(tables, spans)
        positions = np.array([p for a, b in spans for p in range(a, b)]) + 60
        key = torch.empty(k[rows].shape, dtype=k.dtype, device=device)
        out = kv8.rotary_and_cache_kv8(q[rows], k[rows], v[rows], dev[:, 1],
                                       torch.from_numpy(slots).to(device),
                                       torch.from_numpy(positions).to(device), table,
                                       interleaved=interleaved, out_key=key)
        turned = k8.turned(fk[rows], positions, t, interleaved)
        k8.append(turned[None], fv[rows][None], cache[:, 1:2], slots, dtype)
        assert np.array_equal(dev.cpu().numpy(), cache)
        assert np.array_equal(to_bits(key), ko.float_to_bits(turned.astype(np.float64), dtype))
        want = k8.turned(fq[rows], positions, t, interleaved).astype(np.float64)
        assert np.array_equal(to_bits(out), ko.float_to_bits(want, dtype))


def test_a_position_outside_the_table_gives_nan_in_its_own_rows(device):
    rng, (q, k, v), (fq, fk, fv), table, t = _turn_setup(device, 4, 4, 2, 64, 32, "bf16", 5, 10)
    positions = np.array([9, 10, -1, 1 << 40])
    slots = torch.arange(4, device=device) + 16
    pos = torch.from_numpy(positions).to(device)
    kc = torch.zeros(2, 2, 16, 2, 64, dtype=torch.bfloat16, device=device)
    out = rotary.rotary_and_cache(q, k, v, kc[:, 0], kc[:, 1], slots, pos, table)
    for x in (out, kc[1, 0, :4]):
        assert torch.isfinite(x[0]).all() and torch.isnan(x[1:, :, :32].float()).all()
        assert torch.isfinite(x[1:, :, 32:]).all()
    assert torch.isfinite(kc[1, 1]).all()
    cache = np.zeros((2, 1, k8.block_bytes(2, 64)), dtype=np.uint8)
    dev = torch.from_numpy(cache).to(device)
    kv8.rotary_and_cache_kv8(q, k, v, dev[:, 0], slots, pos, table)
    k8.append(k8.turned(fk, positions, t, False)[None], fv[None], cache, np.arange(4) + 16, "bf16")
    assert np.array_equal(dev.cpu().numpy(), cache)


# ---------------------------------------------------------------------------
# de-page
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("H,D", [(1, 64), (4, 128), (2, 256), (11, 128), (5, 64), (9, 256)])
def test_gather_values(device, dtype, H, D):
    rng = np.random.default_rng(H + D)
    lens = np.array([1, 0, 15, 16, 17, 70, 33])
    cache = _filled(rng, 24, 3, H, D, dtype)
    tables = _tables(rng, lens, 24)
    padded = ko.pad_block_tables(tables)
    for layers in (None, (1, 2)):
        k, v = kv8.gather_tokens_kv8(torch.from_numpy(cache).to(device),
                                     torch.from_numpy(padded).to(device),
                                     torch.from_numpy(lens.astype(np.int32)).to(device),
                                     int(lens.sum()), int(lens.max()), D, dtype=DTYPES[dtype],
                                     layers=layers)
        first, count = layers or (0, 3)
        for l in range(count):
            rows = k8.rows(cache[:, first + l], H, D)
            for got, side in ((k, rows[0]), (v, rows[1])):
                want = np.concatenate([side[t].reshape(-1, H, D)[:n] if t else side[:0].reshape(0, H, D)
                                       for t, n in zip(tables, lens)])
                assert np.array_equal(got[l].double().cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_gather_of_every_code_and_exponent(device, dtype, D):
    """Every code under every exponent that the type's rows can have, NaN among
    them."""
    es = np.arange(k8.LOW[dtype], k8.TOP[dtype] + 1)
    n = len(es)
    cache = np.zeros((n, 1, k8.block_bytes(1, D)), dtype=np.uint8)
    rng = np.random.default_rng(D)
    reps = 32 * D // 256
    for i, e in enumerate(es):
        cache[i, 0, :32 * D] = rng.permutation(np.repeat(np.arange(256), reps)).astype(np.uint8)
        cache[i, 0, 32 * D:32 * D + 2] = e + 127
    tables = torch.arange(n, dtype=torch.int32, device=device)[None]
    lens = torch.tensor([16 * n], dtype=torch.int32, device=device)
    got = kv8.gather_tokens_kv8(torch.from_numpy(cache).to(device), tables, lens, 16 * n, 16 * n, D,
                                dtype=DTYPES[dtype])
    for x, want in zip(got, k8.rows(cache[:, 0], 1, D)):
        x = x[0].double().cpu().numpy()
        want = want.reshape(-1, 1, D)
        assert np.array_equal(np.isnan(x), np.isnan(want))
        assert np.array_equal(np.nan_to_num(x), np.nan_to_num(want))


def test_gather_leaves_what_it_is_not_to_write(device):
    """Gaps between the sequences, tokens past the output, unreadable blocks
    and lengths past the bound: those rows stay as they were."""
    rng = np.random.default_rng(1)
    H, D = 2, 64
    cache = torch.from_numpy(_filled(rng, 8, 1, H, D, "bf16")).to(device)
    tables = torch.tensor([[3, 99], [1, -5], [6, 7]], dtype=torch.int32, device=device)
    lens = torch.tensor([20, 18, 1000], dtype=torch.int32, device=device)
    cu = torch.tensor([2, 30, 50, 70], dtype=torch.int32, device=device)
    k, v = kv8.gather_tokens_kv8(cache, tables, lens, 60, 32, D, cu_seqlens=cu)
    for got, want in zip((k, v), k8.rows(cache[:, 0].cpu().numpy(), H, D)):
        got = got[0].double().cpu().numpy()
        assert np.array_equal(got[2:18], want[3])     # 18..21: block 99
        assert np.array_equal(got[30:46], want[1])    # 46, 47: block -5
        assert np.array_equal(got[50:60], want[6][:10])  # cut by the output's end
    out_k, _ = kv8.gather_tokens_kv8(cache, tables, lens, 100, 32, D, cu_seqlens=cu)
    want_k, _ = k8.rows(cache[:, 0].cpu().numpy(), H, D)
    assert np.array_equal(out_k[0, 66:82].double().cpu().numpy(), want_k[7])


def test_gather_batch_past_one_launch(device):
    rng = np.random.default_rng(2)
    lens = rng.integers(0, 20, size=1500)
    cache = _filled(rng, 64, 1, 1, 64, "fp16")
    tables = [[int(x) for x in rng.integers(0, 64, size=-(-n // 16))] for n in lens]
    got = kv8.gather_tokens_kv8(torch.from_numpy(cache).to(device),
                                torch.from_numpy(ko.pad_block_tables(tables)).to(device),
                                torch.from_numpy(lens.astype(np.int32)).to(device),
                                int(lens.sum()), int(lens.max()), 64, dtype=torch.float16)
    for x, side in zip(got, k8.rows(cache[:, 0], 1, 64)):
        want = np.concatenate([side[t].reshape(-1, 1, 64)[:n] for t, n in zip(tables, lens) if n])
        assert np.array_equal(x[0].double().cpu().numpy(), want)


# ---------------------------------------------------------------------------
# other streams, graphs, the block operations, refusals
# ---------------------------------------------------------------------------
def test_captured_appends_replay(device):
    """A captured step replayed with new rows, positions and slots in the same
    tensors equals the eager calls, in either cache."""
    Hq, Hkv, D, T = 28, 4, 128, 16
    rng, (q, k, v), _, table, _ = _turn_setup(device, T, Hq, Hkv, D, D, "bf16", 11)
    slots = torch.arange(T, device=device) * 16
    positions = torch.zeros(T, dtype=torch.int64, device=device)
    c8 = [kv8.kv8_cache(T, 1, Hkv, D, device) for _ in range(2)]
    c16 = [torch.zeros(T, 2, 16, Hkv, D, dtype=torch.bfloat16, device=device) for _ in range(2)]
    outs = [torch.empty(T, Hq, D, dtype=torch.bfloat16, device=device) for _ in range(2)]

    def step(i):
        kv8.rotary_and_cache_kv8(q, k, v, c8[i][:, 0], slots, positions, table, out=outs[i])
        rotary.rotary_and_cache(q, k, v, c16[i][:, 0], c16[i][:, 1], slots, positions, table,
                                out=outs[i])

    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(0)
    for n in range(16):
        q.mul_(-1.1)
        k.mul_(1.3 if n % 3 else -0.4)
        v.mul_(0.8)
        torch.cuda.synchronize()
        g.replay()
        step(1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))
        assert torch.equal(c8[0], c8[1])
        assert torch.equal(c16[0].view(torch.int16), c16[1].view(torch.int16))
        slots += 1
        positions += 1


def test_two_threads_append_to_two_caches(device):
    rng = np.random.default_rng(4)
    H, D, T = 2, 128, 200
    want = []
    caches = [kv8.kv8_cache(16, 1, H, D, device) for _ in range(2)]
    rows = [_rows(rng, (2, 1, T, H, D), "fp16") for _ in range(2)]
    slots = torch.arange(T, device=device)
    for x in rows:
        c = np.zeros((16, 1, k8.block_bytes(H, D)), dtype=np.uint8)
        f = ko.bits_to_float(x, "fp16")
        k8.append(f[0], f[1], c, np.arange(T), "fp16")
        want.append(c)

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            x = to_device_bits(rows[i], "fp16", device)
            for _ in range(20):
                kv8.append_kv8(x[0], x[1], caches[i], slots)
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for c, w in zip(caches, want):
        assert np.array_equal(c.cpu().numpy(), w)


def test_a_larger_pool_past_32_bit_offsets(device):
    """Blocks whose byte offset passes 2^32."""
    H, D, n, layers = 1, 128, 40000, 32  # 135168 bytes per block, 5.4e9 in all
    cache = torch.empty((n, layers, k8.block_bytes(H, D)), dtype=torch.uint8, device=device)
    rng = np.random.default_rng(2)
    tables = [[n - 1, 5, n - 70], [n - 3000]]
    lens = np.array([40, 16])
    slots = _slots(tables, [(0, 40), (0, 16)])
    x = _rows(rng, (2, 56, H, D), "bf16")
    dx = to_device_bits(x, "bf16", device)
    kv8.reshape_and_cache_kv8(dx[0], dx[1], cache[:, 31], torch.from_numpy(slots).to(device))
    bt = torch.from_numpy(ko.pad_block_tables(tables)).to(device)
    sl = torch.from_numpy(lens.astype(np.int32)).to(device)
    got = kv8.gather_tokens_kv8(cache, bt, sl, 56, 40, D, layers=(31, 1))
    small = np.zeros((4, 1, k8.block_bytes(H, D)), dtype=np.uint8)
    f = ko.bits_to_float(x, "bf16")
    at = np.concatenate([np.arange(40), 48 + np.arange(16)])
    k8.append(f[0][None], f[1][None], small, at, "bf16")
    for y, side in zip(got, k8.rows(small[:, 0], H, D)):
        assert np.array_equal(y[0].double().cpu().numpy(), side.reshape(-1, H, D)[at])


def test_the_cache_through_the_block_ops(device):
    """A sequence's life: turned and appended, swapped out to pinned memory and
    back into other blocks, grown by a token, compacted, read."""
    rng = np.random.default_rng(77)
    L, H, D, n = 3, 2, 128, 32
    lens = np.array([70, 33, 16, 5])
    cache = kv8.kv8_cache(n, L, H, D, device)
    tables = _tables(rng, lens + 1, n)
    f = _rows(rng, (2, L, int(lens.sum()) + 4, H, D), "bf16")
    x = to_device_bits(f, "bf16", device)
    m = int(lens.sum())
    kv8.append_kv8(x[0, :, :m], x[1, :, :m], cache,
                   torch.from_numpy(_slots(tables, [(0, a) for a in lens])).to(device))
    used = [b for t in tables for b in t]
    host = torch.empty((len(used), *cache.shape[1:]), dtype=torch.uint8, pin_memory=True)
    ops.swap(used, list(range(len(used))), False, cache, host)
    torch.cuda.synchronize()
    cache.fill_(255)
    new = [int(b) for b in rng.permutation(n)[:len(used)]]
    ops.swap(list(range(len(used))), new, True, cache, host)
    moved = dict(zip(used, new))
    tables = [[moved[b] for b in t] for t in tables]
    kv8.append_kv8(x[0, :, m:], x[1, :, m:], cache,
                   torch.from_numpy(_slots(tables, [(a, a + 1) for a in lens])).to(device))
    from aegaeon_amd.pool import plan_compaction, remap_tables
    src, dst = plan_compaction(new, range(n))
    if len(src):
        ops.defrag_blocks(cache, src, dst)
    tables = remap_tables(tables, src, dst)
    sl = torch.from_numpy((lens + 1).astype(np.int32)).to(device)
    got = kv8.gather_tokens_kv8(cache, torch.from_numpy(ko.pad_block_tables(tables)).to(device), sl,
                                m + 4, int(lens.max()) + 1, D)
    g = ko.bits_to_float(f, "bf16")
    want = np.zeros((n, L, k8.block_bytes(H, D)), dtype=np.uint8)
    k8.append(g[0, :, :m], g[1, :, :m], want, _slots(tables, [(0, a) for a in lens]), "bf16")
    k8.append(g[0, :, m:], g[1, :, m:], want, _slots(tables, [(a, a + 1) for a in lens]), "bf16")
    for l in range(L):
        for y, side in zip(got, k8.rows(want[:, l], H, D)):
            assert np.array_equal(y[l].double().cpu().numpy(), np.concatenate(
                [side[t].reshape(-1, H, D)[:a + 1] for t, a in zip(tables, lens)]))


def test_refusals(device):
    cache = kv8.kv8_cache(4, 2, 4, 128, device)
    x = torch.zeros(2, 3, 4, 128, dtype=torch.bfloat16, device=device)
    slots = torch.zeros(3, dtype=torch.int64, device=device)
    with pytest.raises(ValueError, match="slot"):
        kv8.append_kv8(x, x, cache, slots[:2])
    with pytest.raises(ValueError, match="int64"):
        kv8.append_kv8(x, x, cache, slots.int())
    with pytest.raises(ValueError, match="dtype"):
        kv8.append_kv8(x.float(), x.float(), cache, slots)
    with pytest.raises(ValueError, match="dtype"):
        kv8.append_kv8(x, x.half(), cache, slots)
    with pytest.raises(ValueError, match="layers"):
        kv8.append_kv8(x[:1], x[:1], cache, slots)
    with pytest.raises(ValueError, match="heads"):
        kv8.append_kv8(x[:, :, :2].contiguous(), x[:, :, :2].contiguous(), cache, slots)
    with pytest.raises(ValueError, match="uint8"):
        kv8.append_kv8(x, x, cache.view(torch.int8), slots)
    with pytest.raises(ValueError, match="R = "):
        kv8.append_kv8(x, x, cache[:, :, :-16], slots)
    with pytest.raises(ValueError, match="dense"):
        kv8.append_kv8(x[..., ::2], x[..., ::2], cache, slots)
    bt = torch.zeros(1, 2, dtype=torch.int32, device=device)
    sl = torch.ones(1, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="dtype"):
        kv8.gather_tokens_kv8(cache, bt, sl, 1, 1, 128, dtype=torch.float32)
    with pytest.raises(ValueError, match="R = "):
        kv8.gather_tokens_kv8(kv8.kv8_cache(4, 2, 3, 64, device), bt, sl, 1, 1, 128)
    with pytest.raises(ValueError, match="layer range"):
        kv8.gather_tokens_kv8(cache, bt, sl, 1, 1, 128, layers=(1, 2))
    with pytest.raises(AegkvError):
        kv8.gather_tokens_kv8(cache, bt, sl, 1, 100, 128)


def test_rotary_refusals(device):
    D = 128
    cache = kv8.kv8_cache(4, 1, 2, D, device)
    kc = torch.zeros(4, 2, 16, 2, D, dtype=torch.bfloat16, device=device)
    fused = torch.zeros(3, 12 * D, dtype=torch.bfloat16, device=device)
    q, k, v = (x.unflatten(1, (-1, D)) for x in fused.split([8 * D, 2 * D, 2 * D], 1))
    ids = torch.zeros(3, dtype=torch.int64, device=device)
    table = rotary.rotary_table(8, D, device=device)

    def both(match, q=q, k=k, v=v, slots=ids, pos=ids, table=table, **kw):
        with pytest.raises(ValueError, match=match):
            kv8.rotary_and_cache_kv8(q, k, v, cache[:, 0], slots, pos, table, **kw)
        with pytest.raises(ValueError, match=match):
            rotary.rotary_and_cache(q, k, v, kc[:, 0], kc[:, 1], slots, pos, table, **kw)

    both("positions", pos=ids[:2])
    both("positions", pos=ids.int())
    both("slot_mapping", slots=ids.cpu())
    both("table", table=table.half())
    both("table", table=table[:, ::2])
    both("table", table=rotary.rotary_table(8, 256, device=device))
    both("table", table=table[:0])
    both("dtype", v=v.half())
    both("tokens", k=k[:2], v=v[:2])
    both("out", out=torch.zeros(3, 8, D, dtype=torch.float16, device=device))
    both("out", out=torch.zeros(3, 8, 2 * D, dtype=q.dtype, device=device)[..., :D])
    wide = torch.zeros(4, 8, D, dtype=q.dtype, device=device)
    both("overlaps", q=wide[:3], out=wide[1:])
    both("overlaps", out_key=q[:, 2:4])
    both("overlaps", out_key=v)
    both("overlap each other", out=q[:1].clone().expand(3, -1, -1))
    both("overlap each other", out_key=k[:1].clone().expand(3, -1, -1))
    with pytest.raises(ValueError, match="overlaps"):
        kv8.rotary_and_cache_kv8(q, k, v, cache[:, 0], ids, ids, table, out_key=k)
    with pytest.raises(ValueError, match="heads"):
        kv8.rotary_and_cache_kv8(q, k[:, :1], v[:, :1], cache[:, 0], ids, ids, table)
    with pytest.raises(ValueError, match="matching"):
        rotary.rotary_and_cache(q, k[:, :1], v[:, :1], kc[:, 0], kc[:, 1], ids, ids, table)
    with pytest.raises(ValueError, match="16-bit dtype"):
        rotary.rotary_and_cache(q, k, v, kc[:, 0].half(), kc[:, 1].half(), ids, ids, table)
    with pytest.raises(AegkvError):
        kv8.rotary_and_cache_kv8(q, k, v, cache[:, 0], ids, ids,
                                 torch.zeros(8, 24, device=device))

"""GPU parity of the 8-bit cache's append where a call's rows are not a few prompts:
rows that are skipped between the tokens of a block, and single tokens of many blocks,
which a wave takes four at a time.  Every byte of the cache equals the oracle's."""
from functools import lru_cache

import numpy as np
import pytest
import torch

from aegaeon_amd import kv8, rotary
from oracle import kv8_oracle as k8
from oracle import kv_oracle as ko
from tests.kvtest_utils import to_bits, to_device_bits

pytestmark = pytest.mark.gpu


def _rows(rng, shape, dtype):
    """Rows whose channels and tokens differ much in size, as bits."""
    x = rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[-1])) \
        * np.exp(rng.standard_normal(shape[:-1]))[..., None]
    return ko.float_to_bits(x, dtype)


def _filled(rng, n, layers, heads, dim, dtype):
    """A cache whose every slot was written, as the oracle holds it."""
    cache = np.full((n, layers, k8.block_bytes(heads, dim)), 0xFF, dtype=np.uint8)
    x = ko.bits_to_float(_rows(rng, (2, layers, n * 16, heads, dim), dtype), dtype)
    k8.append(x[0], x[1], cache, np.arange(n * 16), dtype)
    return cache


def _check_append(device, key, value, cache, slots, dtype):
    dev = torch.from_numpy(cache).to(device)
    slots = np.asarray(slots, dtype=np.int64)
    kv8.append_kv8(to_device_bits(key, dtype, device), to_device_bits(value, dtype, device), dev,
                   torch.from_numpy(slots).to(device))
    k8.append(ko.bits_to_float(key, dtype), ko.bits_to_float(value, dtype), cache, slots, dtype)
    assert np.array_equal(dev.cpu().numpy(), cache)


# ---------------------------------------------------------------------------
# skipped rows do not part a block's tokens
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("slots", [
    [16, -1, 17], [17, 4 * 16, 16], [20, -1, -1, 21, -9, 22], [-1, 18, -1, 17, -1, 18, -1],
    [31, -1, 32, -1, 30 - 16, -1, 15, -1, 48]])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_skipped_rows_between_the_tokens_of_a_block(device, slots, dtype):
    rng = np.random.default_rng(len(slots))
    cache = _filled(rng, 4, 2, 3, 128, dtype)
    k, v = (_rows(rng, (2, len(slots), 3, 128), dtype) for _ in range(2))
    _check_append(device, k, v, cache, slots, dtype)


@pytest.mark.parametrize("gap", [1, 20, 30, 46, 47, 62, 63, 64, 65, 511, 512, 513, 575, 576, 1100])
@pytest.mark.parametrize("before", [0, 15])
@pytest.mark.parametrize("heads", [2, 40])
def test_long_gaps(device, gap, before, heads):
    """Gaps of every length about the 64 rows of a wave and the 512 of a search, in
    order and not, behind tokens of another block or none, ended by another block's or
    by the call."""
    rng = np.random.default_rng(gap + before)
    for places, behind in (([3, 4, 5], []), ([0, 9, 2], [33, 34]), ([7, 7], [-1] * 300)):
        slots = [0] * before
        for p in places:
            slots += [16 + p] + [-1] * gap
        slots += behind
        cache = _filled(rng, 3, 1, heads, 64, "bf16")
        k, v = (_rows(rng, (1, len(slots), heads, 64), "bf16") for _ in range(2))
        _check_append(device, k, v, cache, slots, "bf16")


@pytest.mark.parametrize("layers", [1, 9])
def test_a_padded_batch(device, layers):
    """Sequences of a batch padded to one length with skipped rows, single tokens
    and prompts among them, in blocks that begin anywhere."""
    rng = np.random.default_rng(layers)
    lens, width = [1, 3, 40, 1, 17, 1, 1, 64, 2], 70
    slots, block = np.full((len(lens), width), -1), 0
    for b, n in enumerate(lens):
        start = int(rng.integers(0, 16))
        at = rng.permutation(width)[:n] if b % 2 else np.arange(n)  # spread, or to the left
        slots[b, np.sort(at)] = block * 16 + start + np.arange(n)
        block += -(-(start + n) // 16)
    cache = _filled(rng, block, layers, 4, 128, "fp16")
    k, v = (_rows(rng, (layers, slots.size, 4, 128), "fp16") for _ in range(2))
    _check_append(device, k, v, cache, slots.reshape(-1), "fp16")


@pytest.mark.parametrize("interleaved", [False, True])
def test_skipped_rows_of_a_rotating_append(device, interleaved):
    """Drafted tokens of some of a batch's sequences, the others' rows skipped; all
    queries and kept keys are turned."""
    rng = np.random.default_rng(5)
    B, m, Hq, Hkv, D = 40, 4, 4, 2, 64
    slots = np.full((B, m), -1)
    for b in range(B):
        n = int(rng.integers(0, m + 1))
        slots[b, np.sort(rng.permutation(m)[:n])] = b * 16 + int(rng.integers(0, 16 - n)) + np.arange(n)
    slots = slots.reshape(-1)
    x = _rows(rng, (B * m, Hq + 2 * Hkv, D), "bf16")
    q, k, v = (y.contiguous() for y in to_device_bits(x, "bf16", device).split([Hq, Hkv, Hkv], 1))
    f = ko.bits_to_float(x, "bf16")
    positions = rng.integers(0, 100, size=B * m)
    table = rotary.rotary_table(100, D, device=device)
    cache = _filled(rng, B, 1, Hkv, D, "bf16")
    dev = torch.from_numpy(cache).to(device)
    key = torch.empty_like(k)
    out = kv8.rotary_and_cache_kv8(q, k, v, dev[:, 0], torch.from_numpy(slots).to(device),
                                   torch.from_numpy(positions).to(device), table,
                                   interleaved=interleaved, out_key=key)
    turned = [k8.turned(y, positions, table.cpu().numpy(), interleaved)
              for y in (f[:, :Hq], f[:, Hq:Hq + Hkv])]
    k8.append(turned[1][None], f[None, :, Hq + Hkv:], cache, slots, "bf16")
    assert np.array_equal(dev.cpu().numpy(), cache)
    for got, want in ((out, turned[0]), (key, turned[1])):
        assert np.array_equal(to_bits(got), ko.float_to_bits(want.astype(np.float64), "bf16"))


# ---------------------------------------------------------------------------
# decode steps: single tokens, several runs of a wave at once
# ---------------------------------------------------------------------------
def _window(waves):
    """Tokens whose runs a wave takes, of so many (token, head, side, layer)."""
    w = 1
    while w < 16 and waves > 2048 * w:
        w *= 2
    return w


def _windows_of_singles(slots, window, n_slots):
    """The windows in which two tokens or more begin, each the only one of its block."""
    held = [t for t, s in enumerate(slots) if 0 <= s < n_slots]
    block = {t: slots[t] // 16 for t in held}
    begins = [t for i, t in enumerate(held) if i == 0 or block[held[i - 1]] != block[t]]
    alone = {t for t in begins if not any(block.get(x) == block[t] for x in held if x > t)}
    found = 0
    for w in range(0, len(slots), window):
        here = [t for t in begins if w <= t < w + window]
        found += len(here) > 1 and all(t in alone for t in here)
    return found


@lru_cache(maxsize=None)
def _filled_once(n, layers, heads, dim, dtype):
    return _filled(np.random.default_rng(n + heads + dim), n, layers, heads, dim, dtype)


def _steps(rng, T, n_blocks):
    """(slots, gains) of three calls for T sequences: single tokens at any place, a
    tenth skipped; the next place, which may be a block's first; then the next one or
    two.  Gains raise most blocks' exponents in the first call and few later."""
    fresh = [int(b) for b in rng.permutation(n_blocks)]
    at = np.array([fresh.pop() * 16 + int(rng.choice([0, 1, 5, 10, 14, 15])) for _ in range(T)])
    for step in range(3):
        slots = []
        for b in range(T):
            for _ in range(2 if step == 2 and b % 9 == 0 else 1):
                if rng.random() < 0.1:
                    slots.append(int(rng.choice([-1, n_blocks * 16, -50])))
                    continue
                slots.append(int(at[b]))
                at[b] = at[b] + 1 if at[b] % 16 < 15 else fresh.pop() * 16
        gains = 2.0 ** rng.integers(-9 if step else -4, 4 if step else 10, size=len(slots))
        yield np.array(slots, dtype=np.int64), gains


def _scaled(rng, shape, gains, dtype):
    """Rows [.., T, H, D] times their tokens' gains, infinities and NaN in a few."""
    x = ko.bits_to_float(_rows(rng, shape, dtype), dtype) * gains[:, None, None]
    for _ in range(6):
        at = tuple(int(rng.integers(0, n)) for n in shape)
        x[at] = rng.choice([np.inf, -np.inf, np.nan])
    with np.errstate(over="ignore"):
        return ko.float_to_bits(x, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("layers,window", [(2, 2), (4, 4), (8, 8), (16, 16)])
def test_steps_of_single_tokens(device, dtype, D, layers, window):
    """Layers beyond the second take the rows of the first two."""
    T, H, n = 131, 4, 300
    assert _window(2 * layers * H * T) == window
    rng = np.random.default_rng(D + layers)
    cache = _filled_once(n, 2, H, D, dtype).copy()
    dev = torch.from_numpy(cache).to(device).repeat(1, layers // 2, 1)
    for step, (slots, gains) in enumerate(_steps(rng, T, n)):
        # (the third call mixes windows of single tokens and of pairs, as they come)
        assert step == 2 or _windows_of_singles(slots, window, n * 16) > 2
        k, v = (_scaled(rng, (2, len(slots), H, D), gains, dtype) for _ in range(2))
        dk, dv = (to_device_bits(x, dtype, device).repeat(layers // 2, 1, 1, 1) for x in (k, v))
        kv8.append_kv8(dk, dv, dev, torch.from_numpy(slots).to(device))
        k8.append(ko.bits_to_float(k, dtype), ko.bits_to_float(v, dtype), cache, slots, dtype)
        want = torch.from_numpy(cache).to(device).repeat(1, layers // 2, 1)
        assert torch.equal(dev, want), step


def _rotating_step(device, rng, dev, cache, slots, gains, Hq, D, table, dtype, interleaved):
    H, T = (cache.shape[2] // (32 * D)), len(slots)
    q = _scaled(rng, (T, Hq, D), gains, dtype)
    k, v = (_scaled(rng, (T, H, D), gains, dtype) for _ in range(2))
    positions = rng.integers(0, 900, size=T)
    dq, dk, dv = (to_device_bits(x, dtype, device) for x in (q, k, v))
    kv8.rotary_and_cache_kv8(dq, dk, dv, dev[:, 0], torch.from_numpy(slots).to(device),
                             torch.from_numpy(positions).to(device), table, out=dq,
                             interleaved=interleaved)
    t = table.cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        turned = k8.turned(ko.bits_to_float(k, dtype), positions, t, interleaved)
        want_q = k8.turned(ko.bits_to_float(q, dtype), positions, t, interleaved)
        want = ko.bits_to_float(ko.float_to_bits(want_q.astype(np.float64), dtype), dtype)
    k8.append(turned[None], ko.bits_to_float(v, dtype)[None], cache, slots, dtype)
    assert np.array_equal(dev.cpu().numpy(), cache)
    got = dq.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.nan_to_num(got), np.nan_to_num(want))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,rot", [(64, 32), (128, 128), (256, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotating_steps_of_single_tokens(device, dtype, D, rot, interleaved):
    T, H, n = 131, 8, 300
    assert _window(2 * H * T) == 2
    rng = np.random.default_rng(D + rot)
    cache = _filled_once(n, 1, H, D, dtype).copy()
    dev = torch.from_numpy(cache).to(device)
    table = rotary.rotary_table(900, rot, device=device)
    for step, (slots, gains) in enumerate(_steps(rng, T, n)):
        assert _windows_of_singles(slots, 2, n * 16) > 10
        _rotating_step(device, rng, dev, cache, slots, gains, 5, D, table, dtype, interleaved)


@pytest.mark.parametrize("dtype,interleaved", [("bf16", False), ("fp16", True)])
def test_rotating_steps_past_the_largest_window(device, dtype, interleaved):
    T, H, D, n = 210, 40, 128, 300
    assert _window(2 * H * T) == 16
    rng = np.random.default_rng(6)
    cache = np.zeros((n, 1, k8.block_bytes(H, D)), dtype=np.uint8)
    dev = torch.from_numpy(cache).to(device)
    table = rotary.rotary_table(900, D, device=device)
    slots, gains = next(_steps(rng, T, n))
    assert _windows_of_singles(slots, 16, n * 16) > 10
    _rotating_step(device, rng, dev, cache, slots, gains, 40, D, table, dtype, interleaved)


def test_outputs_that_overlap_what_the_call_uses_are_refused(device):
    """Slots, positions, the table and either cache, and nothing was written."""
    T, H, D = 4, 2, 64
    q, k, v = (torch.ones(T, H, D, dtype=torch.float16, device=device) for _ in range(3))
    ids = torch.zeros(64 * T, dtype=torch.int64, device=device)
    table = rotary.rotary_table(8, D, device=device)
    c8 = kv8.kv8_cache(4, 2, H, D, device)
    c16 = torch.zeros(4, 2, 16, H, D, dtype=torch.float16, device=device)

    def rows(x):
        return x.view(torch.float16).reshape(-1)[:T * H * D].view(T, H, D)

    def call(eight, slots=ids[:T], positions=ids[:T], **kw):
        if eight:
            kv8.rotary_and_cache_kv8(q, k, v, c8[:, 1], slots, positions, table, **kw)
        else:
            rotary.rotary_and_cache(q, k, v, c16[:, 0], c16[:, 1], slots, positions, table, **kw)

    before = [x.clone() for x in (ids, table, c8, c16)]
    other = torch.zeros_like(ids)
    for eight in (False, True):
        for name in ("out", "out_key"):
            with pytest.raises(ValueError, match=f"{name} overlaps slot_mapping"):
                call(eight, positions=other[:T], **{name: rows(ids)})
            with pytest.raises(ValueError, match=f"{name} overlaps positions"):
                call(eight, slots=other[:T], **{name: rows(ids)})
            with pytest.raises(ValueError, match=f"{name} overlaps table"):
                call(eight, **{name: rows(table)})
            if eight:
                with pytest.raises(ValueError, match=f"{name} overlaps kv_cache"):
                    call(True, **{name: rows(c8[2, 1])})
            else:
                for side in (0, 1):
                    with pytest.raises(ValueError, match=f"{name} overlaps (key|value)_cache"):
                        call(False, **{name: rows(c16[3, side])})
    for x, y in zip((ids, table, c8, c16), before):
        assert torch.equal(x, y)
    whole = torch.zeros(3 * T * H * D, dtype=torch.float16, device=device)  # touching is clear
    a, b, c = whole.view(3, T, H, D)
    rotary.rotary_and_cache(b, k, v, c16[:, 0], c16[:, 1], ids[:T], ids[:T], table, out=a, out_key=c)

"""The 4-bit KV cache without a GPU: the oracle's numbers and bytes pinned by
hand, and the refusals of the C ABI and of the Python entry points."""
import numpy as np
import pytest
import torch

from aegaeon_amd import _lib, kv4
from oracle import kv4_oracle as k4
from oracle import kv_oracle as ko

OK, INVALID, MISALIGNED, UNSUP, WS = 0, -1, -3, -6, -7


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------
def _group(*head):
    x = np.zeros(32)
    x[:len(head)] = head
    return x


@pytest.mark.parametrize("head,scale,codes", [
    ((6.0,), 127, [7]),                       # 6 < 7 * 2^0
    ((6.9999,), 127, [7]),                    # rounds to 6
    ((7.0,), 128, [6]),                       # the next exponent: 3.5 is midway, to the even code 4
    ((3.5,), 127, [6]),                       # 3.5 < 7 * 2^-1 fails: e = 0, 3.5 -> code of 4
    ((3.4999,), 126, [7]),                    # 6.9998 -> 6
    ((4.0, 0.25, -0.25, 0.75, 1.25, 1.75, 2.5, -5.0), 127, [6, 0, 8, 2, 2, 4, 4, 14]),  # ties
    ((4.0, 0.26, 0.74, 1.26, 1.74, 2.51, 3.49), 127, [6, 1, 1, 3, 3, 5, 5]),
    ((0.0, -0.0), 2, [0, 8]),
    ((1e-45,), 2, [0]),                       # below half a step of the least scale
    ((2.0 ** -126,), 2, [1]),
])
def test_group_codes_by_hand(head, scale, codes):
    c, s = k4.encode(_group(*head), "bf16")
    assert s[0] == scale
    assert list(c[:len(codes)]) == codes


def test_largest_values_stay_finite_in_their_type():
    big = 2.0 ** 127 * (2 - 2.0 ** -7)  # the largest bf16
    c, s = k4.encode(_group(big), "bf16")
    assert (c[0], s[0]) == (7, 252)
    assert k4.decode(c, s)[0] == 6 * 2.0 ** 125
    c, s = k4.encode(_group(65504.0, -57344.0), "fp16")
    assert (c[0], c[1], s[0]) == (7, 15, 140)
    assert k4.decode(c, s)[0] == 49152.0
    # 2^14 * 3.4999 still has an exponent of its own
    c, s = k4.encode(_group(57343.0), "fp16")
    assert (c[0], s[0]) == (7, 140)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_group_with_a_non_finite_value_reads_as_nan(bad):
    x = np.zeros(64)
    x[40] = bad
    x[0] = 1.5
    c, s = k4.encode(x, "bf16")
    assert s[1] == 255 and not c[32:].any()
    v = k4.decode(c, s)
    assert v[0] == 1.5 and np.isnan(v[32:]).all() and np.isfinite(v[:32]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_stored_values_are_exact_in_their_type_and_encode_to_themselves(dtype):
    rng = np.random.default_rng(3)
    bits = rng.integers(0, 1 << 16, size=(512, 32)).astype(np.uint16)
    bits[:256] = np.sort(bits[:256].reshape(-1)).reshape(256, 32)
    x = ko.bits_to_float(bits, dtype)
    x = x[np.isfinite(x).all(-1)]
    c, s = k4.encode(x, dtype)
    v = k4.decode(c, s)
    assert np.array_equal(ko.bits_to_float(ko.float_to_bits(v, dtype), dtype), v)
    c2, s2 = k4.encode(v, dtype)
    assert np.array_equal(k4.decode(c2, s2), v)
    # no element further off than half a step of the largest one's binade
    e = s.astype(int) - 127
    capped = s == (252 if dtype == "bf16" else 140)
    off = np.abs(v - x).max(-1)
    assert (off <= np.ldexp(1.0, e[:, 0]))[~capped[:, 0]].all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("side", [0, 1])
def test_every_half_byte_of_a_record_is_one_value(dim, side):
    seen, scales = set(), set()
    for r in range(16):
        for d in range(dim):
            at, half, sc = k4.byte_of(side, dim, r, d)
            assert 0 <= at < 8 * dim and (at, half) not in seen
            seen.add((at, half))
            scales.add(sc)
    assert len(seen) == 16 * dim
    assert scales == set(range(8 * dim, k4.record_bytes(dim)))


@pytest.mark.parametrize("side,dim,r,d,want", [
    (0, 128, 0, 0, (0, 0, 1024)), (0, 128, 5, 31, (95, 1, 1029)), (0, 128, 5, 32, (336, 0, 1045)),
    (0, 64, 3, 17, (152, 1, 515)), (0, 256, 15, 255, (2047, 1, 2175)),
    (1, 128, 0, 8, (16, 0, 1024)), (1, 128, 6, 127, (507, 1, 1078)),
    (1, 64, 2, 5, (12, 1, 514)), (1, 256, 1, 24, (1044, 0, 2049)), (1, 256, 15, 255, (2047, 1, 2175)),
])
def test_byte_positions_by_hand(side, dim, r, d, want):
    assert k4.byte_of(side, dim, r, d) == want


def test_append_then_rows_is_the_identity_on_stored_values():
    rng = np.random.default_rng(0)
    cache = np.full((4, 2, 3, 2, k4.record_bytes(64)), 0xA5, dtype=np.uint8)
    before = cache.copy()
    slots = np.array([0, 17, 63, 64, -1, 5])
    x = ko.bits_to_float(ko.float_to_bits(rng.standard_normal((2, 2, 6, 3, 64)), "bf16"), "bf16")
    k4.append(x[0], x[1], cache, slots, "bf16")
    for layer in range(2):
        got = k4.rows(cache[:, layer], 64)
        for side in (0, 1):
            want = k4.decode(*k4.encode(x[side, layer], "bf16"))
            for t, s in enumerate(slots):
                if 0 <= s < 64:
                    assert np.array_equal(got[side][s // 16, s % 16], want[t])
    assert np.array_equal(cache[2], before[2])


@pytest.mark.parametrize("causal", [True, False])
def test_textbook_attention_is_torchs_in_64_bits(causal):
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((2, 6, 16, 2, 64))
    tables, new, lens = [[3, 1, 0], [5], [4, 2]], [7, 3, 32], [40, 3, 32]
    cu = np.concatenate([[0], np.cumsum(new)])
    q = rng.standard_normal((cu[-1], 6, 64))
    got = k4.varlen_attention(q, k, v, tables, cu, lens, 0.2, causal)
    for b, (m, n) in enumerate(zip(new, lens)):
        mine = slice(cu[b], cu[b + 1])
        rows = [torch.from_numpy(x[tables[b]].reshape(-1, 2, 64)[:n]).transpose(0, 1)
                .repeat_interleave(3, 0) for x in (k, v)]
        seen = torch.ones(m, n, dtype=torch.bool).tril(n - m) if causal else None
        want = torch.nn.functional.scaled_dot_product_attention(
            torch.from_numpy(q[mine]).transpose(0, 1), *rows, attn_mask=seen, scale=0.2)
        assert np.allclose(got[mine], want.transpose(0, 1).numpy(), rtol=1e-12, atol=1e-12)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _buf(nbytes, misalign=0):
    raw = np.zeros(nbytes + 64, dtype=np.uint8)
    return raw, (raw.ctypes.data + 15) // 16 * 16 + misalign


def test_block_bytes(lib):
    assert lib.aegkv_kv4_block_bytes(4, 128) == 4 * 17 * 128
    assert lib.aegkv_kv4_block_bytes(1, 64) == 17 * 64
    assert lib.aegkv_kv4_block_bytes(0, 128) == INVALID
    assert lib.aegkv_kv4_block_bytes(4, 96) == UNSUP
    for d in (64, 128, 256):
        assert kv4.kv4_record_bytes(d) * 2 == lib.aegkv_kv4_block_bytes(1, d)
        assert kv4.kv4_record_bytes(d) == k4.record_bytes(d)
    with pytest.raises(ValueError):
        kv4.kv4_record_bytes(80)


def test_append_host_checks(lib):
    raw, p = _buf(1 << 12)

    def call(key=p, value=p, slots=p, cache=p, n_tokens=4, layers=1, heads=2, dim=64, dt=0, ts=128,
             ls=0, bs=4352, cls=0, blocks=4):
        return lib.aegkv_kv4_append(key, value, ts, 128, ls, 0, slots, n_tokens, cache, bs, cls,
                                    blocks, layers, heads, dim, dt, None)

    assert call(n_tokens=-1) == INVALID
    assert call(layers=0) == INVALID
    assert call(heads=0) == INVALID
    assert call(blocks=-1) == INVALID
    assert call(dim=96) == UNSUP
    assert call(dt=2) == UNSUP
    assert call(n_tokens=0) == OK and call(blocks=0) == OK
    assert call(key=None) == INVALID and call(slots=None) == INVALID and call(cache=None) == INVALID
    assert call(key=p + 2) == MISALIGNED and call(cache=p + 8) == MISALIGNED
    assert call(ts=132) == MISALIGNED and call(ls=4) == MISALIGNED
    assert call(bs=4360) == MISALIGNED and call(cls=8) == MISALIGNED
    assert call(n_tokens=1 << 62) == UNSUP  # no product may wrap
    assert call(n_tokens=1 << 27, heads=2, dim=64) == UNSUP  # 2^32 threads


def test_gather_host_checks(lib):
    raw, p = _buf(1 << 12)

    def call(cache=p, tables=p, out=p, max_blocks=3, batch=2, longest=40, tokens=80, layers=1,
             heads=2, dim=64, dt=0, bs=4352, ols=0):
        return lib.aegkv_kv4_gather_tokens(cache, bs, 0, 4, tables, max_blocks, p, p, batch,
                                           longest, out, p, tokens, ols, layers, heads, dim, dt,
                                           None)

    assert call(max_blocks=2) == INVALID  # 40 tokens need three blocks
    assert call(dim=32) == UNSUP and call(dt=7) == UNSUP
    assert call(batch=-1) == INVALID and call(layers=0) == INVALID and call(heads=-1) == INVALID
    assert call(batch=0, tables=None) == OK and call(longest=0) == OK and call(tokens=0) == OK
    assert call(tables=None) == INVALID and call(out=None) == INVALID
    assert call(out=p + 4) == MISALIGNED and call(bs=17) == MISALIGNED
    assert call(ols=4) == MISALIGNED
    assert call(heads=1 << 24) == UNSUP  # chunks of a block past 32 bits


def test_decode_host_checks(lib):
    raw, p = _buf(1 << 16)

    def attn(hq=28, hkv=4, d=128, dt=0, longest=64, max_blocks=4, ws=p, wsb=1 << 30, nwg=8, q=p,
             cache=p, bs=17 * 4 * 128, tables=p, blocks=8):
        return lib.aegkv_kv4_decode_attention(p, hq * d, q, hq * d, cache, bs, blocks, tables,
                                              max_blocks, p, 2, longest, hq, hkv, d, 0.1, dt, nwg,
                                              ws, wsb, None)

    assert attn(hq=30) == INVALID and attn(d=96) == UNSUP and attn(dt=7) == UNSUP
    assert attn(hq=34, hkv=2) == UNSUP       # 17 query heads per kv head
    assert attn(longest=100) == INVALID      # needs 7 blocks, the table has 4
    assert attn(nwg=-1) == INVALID and attn(nwg=8193) == UNSUP
    assert attn(cache=None) == INVALID and attn(tables=None) == INVALID and attn(blocks=0) == INVALID
    assert attn(q=p + 2) == MISALIGNED and attn(cache=p + 8) == MISALIGNED
    assert attn(bs=17 * 4 * 128 + 8) == MISALIGNED
    need = lib.aegkv_paged_decode_attention_workspace_size(2, 28, 4, 128, 64, 0, 8)
    assert attn(ws=None) == WS and attn(wsb=need - 1) == WS

    def planned(plan=p, nbytes=1 << 16, bs=17 * 4 * 128):
        return lib.aegkv_kv4_decode_attention_planned(p, 28 * 128, p, 28 * 128, p, bs, 8, plan,
                                                      nbytes, p, 2, 64, 28, 4, 128, 0.1, 0, 8, p,
                                                      1 << 30, None)

    assert planned(plan=None) == INVALID
    size = lib.aegkv_paged_decode_plan_size(2, 4, 64, 8)
    assert planned(nbytes=size - 1) == INVALID
    assert planned(bs=8) == MISALIGNED


def test_varlen_host_checks(lib):
    raw, p = _buf(1 << 12)

    def call(out=p, q=p, cache=p, tables=p, cu=p, qs=28 * 128, os_=28 * 128, bs=17 * 512, blocks=8,
             max_blocks=4, batch=1, total=16, max_q=16, longest=64, hq=28, hkv=4, d=128, scale=0.1,
             dt=0, ws=p, wsb=1 << 40):
        return lib.aegkv_kv4_varlen_attention(out, os_, q, qs, cache, bs, blocks, tables, max_blocks,
                                              cu, p, batch, total, max_q, longest, hq, hkv, d,
                                              scale, 1, dt, ws, wsb, None)

    assert call(hkv=5) == INVALID                  # Hq not a multiple of Hkv
    assert call(d=256) == UNSUP and call(d=32) == UNSUP and call(dt=7) == UNSUP
    assert call(scale=float("nan")) == INVALID and call(scale=float("inf")) == INVALID
    assert call(scale=3e38) == INVALID             # infinite times log2 e
    assert call(batch=-1) == INVALID and call(longest=-1) == INVALID and call(max_q=-1) == INVALID
    assert call(batch=0, q=None) == OK and call(total=0) == OK and call(max_q=0) == OK
    assert call(q=None) == INVALID and call(cache=None) == INVALID and call(tables=None) == INVALID
    assert call(cu=None) == INVALID and call(blocks=0) == INVALID
    assert call(qs=27 * 128) == INVALID and call(os_=27 * 128) == INVALID
    assert call(q=p + 2) == MISALIGNED and call(os_=28 * 128 + 4) == MISALIGNED
    assert call(bs=17 * 512 + 8) == MISALIGNED
    assert call(longest=65) == INVALID             # five blocks, the table has four
    assert call(max_q=1 << 30) == UNSUP            # rows past 32 bits
    size = lib.aegkv_kv4_varlen_attention_workspace_size
    assert size(0, 0, 0, 64, 28, 4, 128, 0) == 0
    assert size(1, 16, 16, 64, 28, 5, 128, 0) == INVALID
    assert size(1, 16, 16, 64, 28, 4, 256, 0) == UNSUP


def test_python_entry_points_refuse_host_tensors():
    cache = kv4.kv4_cache(3, 2, 4, 128, device="cpu")
    assert cache.shape == (3, 2, 4, 2, 1088) and not cache.any()
    x = torch.zeros(2, 5, 4, 128, dtype=torch.bfloat16)
    slots = torch.zeros(5, dtype=torch.int64)
    with pytest.raises(ValueError):
        kv4.append_kv4(x, x, cache, slots)
    with pytest.raises(ValueError):
        kv4.reshape_and_cache_kv4(x[0], x[0], cache[:, 0], slots)
    with pytest.raises(ValueError):
        kv4.gather_tokens_kv4(cache, torch.zeros(1, 1, dtype=torch.int32),
                              torch.ones(1, dtype=torch.int32), 1, 1)
    with pytest.raises(ValueError):
        kv4.paged_decode_attention_kv4(x[0], cache[:, 0], torch.zeros(5, 1, dtype=torch.int32),
                                       torch.ones(5, dtype=torch.int32), 0.1, 1)
    with pytest.raises(ValueError):
        kv4.varlen_attention_kv4(x[0], cache[:, 0], torch.zeros(1, 1, dtype=torch.int32),
                                 torch.zeros(2, dtype=torch.int32),
                                 torch.ones(1, dtype=torch.int32), 1, 1, 0.1)

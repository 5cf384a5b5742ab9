"""The 8-bit KV cache and the rotating appends without a GPU: the oracle's numbers
and bytes pinned by hand, and the refusals of the C ABI and of the Python entry
points."""
import numpy as np
import pytest
import torch

from aegaeon_amd import _lib, kv8, rotary
from oracle import kv8_oracle as k8
from oracle import kv_oracle as ko

OK, INVALID, MISALIGNED, UNSUP, WS = 0, -1, -3, -6, -7


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------
def test_codes_are_the_8_bit_floats():
    """Every code's value, and torch's rounding to the same type."""
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).double().numpy()
    got = k8.decode(codes, 0)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(got).sum() == 2
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(20000) * np.exp(4 * rng.standard_normal(20000)),
                        (k8.GRID[1:] + k8.GRID[:-1]) / 2, k8.GRID, -k8.GRID])
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(k8.encode(x, 0), want)


@pytest.mark.parametrize("largest,dtype,e", [
    (448.0, "bf16", 0), (448.0001, "bf16", 1), (224.0, "bf16", -1), (1.0, "bf16", -8),
    (1.75, "bf16", -8), (1.7501, "bf16", -7), (0.0, "bf16", -117), (0.0, "fp16", -15),
    (1e-6, "fp16", -15), (65504.0, "fp16", 7), (57344.0, "fp16", 7), (3.39e38, "bf16", 119)])
def test_exponents_by_hand(largest, dtype, e):
    assert k8.exponent(np.array([0.0, -largest, np.nan, np.inf]), dtype) == e


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_stored_values_are_exact_in_their_type_and_encode_to_themselves(dtype):
    codes = np.array([c for c in range(256) if c & 0x7F != 0x7F], dtype=np.uint8)
    for e in (k8.LOW[dtype], k8.LOW[dtype] + 1, -3, 0, 5, k8.TOP[dtype]):
        v = k8.decode(codes, e)
        assert np.isfinite(v).all()
        assert np.array_equal(ko.bits_to_float(ko.float_to_bits(v, dtype), dtype), v)
        assert np.array_equal(k8.encode(v, e), codes)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("side", [0, 1])
def test_every_byte_of_a_side_is_one_value(dim, side):
    seen = {k8.byte_of(side, dim, r, d) for r in range(16) for d in range(dim)}
    assert seen == set(range(16 * dim))


@pytest.mark.parametrize("side,dim,r,d,want", [
    (0, 128, 0, 0, 0), (0, 128, 5, 15, 95), (0, 128, 5, 16, 336), (0, 64, 15, 63, 1023),
    (1, 128, 0, 8, 16), (1, 128, 6, 4, 1282), (1, 128, 15, 127, 2047), (1, 64, 2, 5, 22),
    (1, 256, 1, 24, 2065)])
def test_byte_positions_by_hand(side, dim, r, d, want):
    assert k8.byte_of(side, dim, r, d) == want


def _one(layer, side, h, heads, dim):
    """(values [16, D], exponent) of a block's side."""
    k = k8.rows(layer[None], heads, dim)[side][0, :, h]
    return k, int(layer[32 * heads * dim + 4 * h + side]) - 127


def test_joining_tokens_raise_the_exponent_and_round_the_earlier_ones_once_more():
    D, cache = 64, np.full((2, 1, k8.block_bytes(1, 64)), 0xEE, dtype=np.uint8)
    x = np.zeros((1, 1, 1, D))
    x[..., 0], x[..., 1] = 1.0, 2.0 ** -16 * 1.125
    k8.append(x, x, cache, np.array([16]), "bf16")        # begins block 1
    v, e = _one(cache[1, 0], 0, 0, 1, D)
    assert e == -8 and v[0, 0] == 1.0 and v[0, 1] == 2.0 ** -16  # 2.25 least steps: 2
    assert not v[1:].any()
    y = np.zeros((1, 1, 1, D))
    y[..., 2] = 0.5
    k8.append(y, y, cache, np.array([18]), "bf16")        # smaller: the exponent stays
    v, e = _one(cache[1, 0], 1, 0, 1, D)
    assert e == -8 and v[0, 0] == 1.0 and v[2, 2] == 0.5
    y[..., 2] = -100.0
    k8.append(y, y, cache, np.array([17]), "bf16")        # 100 <= 448 * 2^-2
    v, e = _one(cache[1, 0], 0, 0, 1, D)
    assert e == -2 and v[0, 0] == 1.0 and v[1, 2] == -96.0  # 400 is midway: the even code's 384
    assert v[0, 1] == 0.0 and v[2, 2] == 0.5              # 2^-16 is below half of 2^-11
    k8.append(x, x, cache, np.array([16]), "bf16")        # and begins it anew
    v, e = _one(cache[1, 0], 0, 0, 1, D)
    assert e == -8 and v[0, 0] == 1.0 and not v[1:].any()
    assert (cache[0] == 0xEE).all()


def test_non_finite_values_are_nan_alone_and_do_not_raise_the_exponent():
    D, cache = 64, np.zeros((1, 1, k8.block_bytes(1, 64)), dtype=np.uint8)
    x = np.ones((1, 2, 1, D))
    x[0, 1, 0, :3] = np.inf, -np.inf, np.nan
    k8.append(x, x, cache, np.array([0, 1]), "fp16")
    v, e = _one(cache[0, 0], 1, 0, 1, D)
    assert e == -8 and np.isnan(v[1, :3]).all() and (v[1, 3:] == 1).all() and (v[0] == 1).all()
    assert cache[0, 0, 32 * D + 2] == 1
    k8.append(x[:, :1], x[:, :1], cache, np.array([5]), "fp16")
    assert cache[0, 0, 32 * D + 2] == 1
    k8.append(x[:, :1], x[:, :1], cache, np.array([0]), "fp16")
    assert cache[0, 0, 32 * D + 2] == 0


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_a_product_of_complex_numbers(interleaved):
    rng = np.random.default_rng(1)
    table = rotary.rotary_table(300, 32, device="cpu").numpy()
    x = rng.standard_normal((5, 2, 64))
    pos = np.array([0, 1, 299, 17, 300])
    got = k8.turned(x, pos, table, interleaved)
    i = np.arange(16)
    turn = np.exp(1j * pos[:, None] * 10000.0 ** (-i / 16))[:, None]
    a, b = (x[..., 0:32:2], x[..., 1:32:2]) if interleaved else (x[..., :16], x[..., 16:32])
    z = (a + 1j * b) * turn
    u, w = (got[..., 0:32:2], got[..., 1:32:2]) if interleaved else (got[..., :16], got[..., 16:32])
    # inputs, table and three operations in float32
    assert np.abs(u - z.real)[:4].max() < 1e-6 and np.abs(w - z.imag)[:4].max() < 1e-6
    assert np.array_equal(got[..., 32:], x[..., 32:].astype(np.float32))
    assert np.isnan(got[4, :, :32]).all()
    assert np.array_equal(got[0], x[0].astype(np.float32))  # position 0 turns nothing


def test_rotary_table_by_hand():
    t = rotary.rotary_table(3, 16, base=100.0, device="cpu")
    assert t.shape == (3, 16) and t.dtype == torch.float32
    angle = 2 * 100.0 ** (-2 * 3 / 16)
    assert t[2, 3] == np.float32(np.cos(angle)) and t[2, 11] == np.float32(np.sin(angle))
    assert (t[0, :8] == 1).all() and (t[0, 8:] == 0).all()
    for bad in (0, -16, 24):
        with pytest.raises(ValueError):
            rotary.rotary_table(3, bad, device="cpu")


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
    assert lib.aegkv_kv8_block_bytes(4, 128) == 4 * 4096 + 128
    assert lib.aegkv_kv8_block_bytes(1, 64) == 2048 + 128
    assert lib.aegkv_kv8_block_bytes(33, 256) == 33 * 8192 + 256
    assert lib.aegkv_kv8_block_bytes(0, 128) == INVALID
    assert lib.aegkv_kv8_block_bytes(4, 96) == UNSUP and lib.aegkv_kv8_block_bytes(257, 64) == UNSUP
    for h in (1, 7, 32, 33, 256):
        for d in (64, 128, 256):
            assert kv8.kv8_block_bytes(h, d) == lib.aegkv_kv8_block_bytes(h, d) \
                == k8.block_bytes(h, d)
            assert kv8.kv8_block_bytes(h, d) // (32 * d) == h  # how a call finds the heads
    for h, d in ((0, 64), (257, 64), (4, 80)):
        with pytest.raises(ValueError):
            kv8.kv8_block_bytes(h, d)


def test_append_host_checks(lib):
    raw, p = _buf(1 << 12)

    def call(key=p, value=p, slots=p, cache=p, n_tokens=4, layers=1, heads=2, dim=64, dt=0, ts=128,
             ls=0, bs=4224, cls=0, blocks=4):
        return lib.aegkv_kv8_append(key, value, ts, 128, ls, 0, slots, n_tokens, cache, bs, cls,
                                    blocks, layers, heads, dim, dt, None)

    assert call(n_tokens=-1) == INVALID and call(layers=0) == INVALID
    assert call(heads=0) == INVALID and call(blocks=-1) == INVALID
    assert call(dim=96) == UNSUP and call(dt=2) == UNSUP and call(heads=257) == UNSUP
    assert call(blocks=1 << 31) == UNSUP
    assert call(n_tokens=0) == OK and call(blocks=0) == OK
    assert call(key=None) == INVALID and call(slots=None) == INVALID and call(cache=None) == INVALID
    assert call(key=p + 2) == MISALIGNED and call(cache=p + 8) == MISALIGNED
    assert call(ts=132) == MISALIGNED and call(ls=4) == MISALIGNED
    assert call(bs=4232) == MISALIGNED and call(cls=8) == MISALIGNED
    assert call(n_tokens=1 << 62) == UNSUP  # no product may wrap
    assert call(n_tokens=1 << 29) == UNSUP  # 2^31 waves


@pytest.mark.parametrize("eight", [False, True])
def test_rotary_append_host_checks(lib, eight):
    raw, p = _buf(1 << 12)

    def call(q=p, oq=p, key=p, value=p, okey=None, slots=p, pos=p, table=p, cache=p, hq=4, hkv=2,
             dim=64, qs=256, oqs=256, ks=128, vs=128, oks=128, n=4, max_pos=8, rot=64, bs=4224,
             blocks=4, block=16, dt=0):
        head = (q, qs, oq, oqs, hq, key, ks, value, vs, okey, oks, hkv, dim, slots, pos, n, table,
                max_pos, rot, 0)
        if eight:
            return lib.aegkv_kv8_rotary_append(*head, cache, bs, blocks, dt, None)
        return lib.aegkv_rotary_append(*head, cache, cache, bs, blocks, block, dt, None)

    assert call(n=-1) == INVALID and call(hq=0) == INVALID and call(hkv=0) == INVALID
    assert call(blocks=-1) == INVALID and call(max_pos=-1) == INVALID
    assert call(rot=0) == INVALID and call(rot=80) == INVALID      # past the head
    assert call(rot=24) == UNSUP and call(dt=2) == UNSUP and call(hq=70000) == UNSUP
    assert call(dim=36, rot=16) == UNSUP
    assert call(n=0, q=None) == OK
    for name in ("q", "oq", "key", "value", "slots", "pos", "table", "cache"):
        assert call(**{name: None}) == INVALID, name
    assert call(max_pos=0) == INVALID
    for name in ("q", "oq", "key", "value", "okey", "table", "cache"):
        assert call(**{name: p + 8}) == MISALIGNED, name
    for name in ("qs", "oqs", "ks", "vs", "oks"):
        assert call(**{name: 132}) == MISALIGNED, name
    assert call(bs=4228) == MISALIGNED
    assert call(n=1 << 31) == UNSUP and call(n=1 << 62) == UNSUP
    if not eight:
        assert call(block=0) == INVALID and call(dim=1024) == UNSUP


def test_gather_host_checks(lib):
    raw, p = _buf(1 << 12)

    def call(cache=p, tables=p, out=p, max_blocks=3, batch=2, longest=40, tokens=80, layers=1,
             heads=2, dim=64, dt=0, bs=4224, ols=0):
        return lib.aegkv_kv8_gather_tokens(cache, bs, 0, 4, tables, max_blocks, p, p, batch,
                                           longest, out, p, tokens, ols, layers, heads, dim, dt,
                                           None)

    assert call(max_blocks=2) == INVALID  # 40 tokens need three blocks
    assert call(dim=32) == UNSUP and call(dt=7) == UNSUP and call(heads=300) == UNSUP
    assert call(batch=-1) == INVALID and call(layers=0) == INVALID and call(heads=-1) == INVALID
    assert call(batch=0, tables=None) == OK and call(longest=0) == OK and call(tokens=0) == OK
    assert call(tables=None) == INVALID and call(out=None) == INVALID
    assert call(out=p + 4) == MISALIGNED and call(bs=17) == MISALIGNED
    assert call(ols=4) == MISALIGNED and call(layers=70000) == UNSUP
    assert call(longest=1 << 30, max_blocks=1 << 27) == UNSUP  # tiles past 32 bits


def test_decode_host_checks(lib):
    raw, p = _buf(1 << 16)

    def attn(hq=28, hkv=4, d=128, dt=0, longest=64, max_blocks=4, ws=p, wsb=1 << 30, nwg=8, q=p,
             cache=p, bs=16512, tables=p, blocks=8, scale=0.1):
        return lib.aegkv_kv8_decode_attention(p, hq * d, q, hq * d, cache, bs, blocks, tables,
                                              max_blocks, p, 2, longest, hq, hkv, d, scale, dt,
                                              nwg, ws, wsb, None)

    assert attn(hq=30) == INVALID and attn(d=96) == UNSUP and attn(dt=7) == UNSUP
    assert attn(hq=34, hkv=2) == UNSUP       # 17 query heads per kv head
    assert attn(hq=257, hkv=257, d=64) == UNSUP
    assert attn(longest=100) == INVALID      # needs 7 blocks, the table has 4
    assert attn(nwg=-1) == INVALID and attn(nwg=8193) == UNSUP
    assert attn(cache=None) == INVALID and attn(tables=None) == INVALID and attn(blocks=0) == INVALID
    assert attn(q=p + 2) == MISALIGNED and attn(cache=p + 8) == MISALIGNED
    assert attn(bs=16520) == MISALIGNED
    for bad in (float("nan"), float("inf"), 3e38):
        assert attn(scale=bad) == INVALID
    need = lib.aegkv_paged_decode_attention_workspace_size(2, 28, 4, 128, 64, 0, 8)
    assert attn(ws=None) == WS and attn(wsb=need - 1) == WS

    def planned(plan=p, nbytes=1 << 16, bs=16512):
        return lib.aegkv_kv8_decode_attention_planned(p, 28 * 128, p, 28 * 128, p, bs, 8, plan,
                                                      nbytes, p, 2, 64, 28, 4, 128, 0.1, 0, 8, p,
                                                      1 << 30, None)

    assert planned(plan=None) == INVALID
    size = lib.aegkv_paged_decode_plan_size(2, 4, 64, 8)
    assert planned(nbytes=size - 1) == INVALID
    assert planned(bs=8) == MISALIGNED


def test_varlen_host_checks(lib):
    raw, p = _buf(1 << 12)

    def call(out=p, q=p, cache=p, tables=p, cu=p, qs=28 * 128, os_=28 * 128, bs=16512, blocks=8,
             max_blocks=4, batch=1, total=16, max_q=16, longest=64, hq=28, hkv=4, d=128, scale=0.1,
             dt=0, ws=p, wsb=1 << 40):
        return lib.aegkv_kv8_varlen_attention(out, os_, q, qs, cache, bs, blocks, tables, max_blocks,
                                              cu, p, batch, total, max_q, longest, hq, hkv, d,
                                              scale, 1, dt, ws, wsb, None)

    assert call(hkv=5) == INVALID                  # Hq not a multiple of Hkv
    assert call(d=256) == UNSUP and call(d=32) == UNSUP and call(dt=7) == UNSUP
    assert call(hq=257, hkv=257) == UNSUP
    assert call(scale=float("nan")) == INVALID and call(scale=float("inf")) == INVALID
    assert call(scale=3e38) == INVALID             # infinite times log2 e
    assert call(batch=-1) == INVALID and call(longest=-1) == INVALID and call(max_q=-1) == INVALID
    assert call(batch=0, q=None) == OK and call(total=0) == OK and call(max_q=0) == OK
    assert call(q=None) == INVALID and call(cache=None) == INVALID and call(tables=None) == INVALID
    assert call(cu=None) == INVALID and call(blocks=0) == INVALID
    assert call(qs=27 * 128) == INVALID and call(os_=27 * 128) == INVALID
    assert call(q=p + 2) == MISALIGNED and call(os_=28 * 128 + 4) == MISALIGNED
    assert call(bs=16520) == MISALIGNED
    assert call(longest=65) == INVALID             # five blocks, the table has four
    assert call(max_q=1 << 30) == UNSUP            # rows past 32 bits
    size = lib.aegkv_kv8_varlen_attention_workspace_size
    assert size(0, 0, 0, 64, 28, 4, 128, 0) == 0
    assert size(1, 16, 16, 64, 28, 5, 128, 0) == INVALID
    assert size(1, 16, 16, 64, 28, 4, 256, 0) == UNSUP
    assert size(1, 16, 16, 64, 257, 257, 64, 0) == UNSUP


def test_python_entry_points_refuse_host_tensors():
    cache = kv8.kv8_cache(3, 2, 4, 128, device="cpu")
    assert cache.shape == (3, 2, 16512) and not cache.any()
    x = torch.zeros(2, 5, 4, 128, dtype=torch.bfloat16)
    slots = torch.zeros(5, dtype=torch.int64)
    table = rotary.rotary_table(8, 128, device="cpu")
    with pytest.raises(ValueError):
        kv8.append_kv8(x, x, cache, slots)
    with pytest.raises(ValueError):
        kv8.reshape_and_cache_kv8(x[0], x[0], cache[:, 0], slots)
    with pytest.raises(ValueError):
        kv8.rotary_and_cache_kv8(x[0], x[0], x[0], cache[:, 0], slots, slots, table)
    with pytest.raises(ValueError):
        rotary.rotary_and_cache(x[0], x[0], x[0], x, x, slots, slots, table)
    with pytest.raises(ValueError):
        kv8.gather_tokens_kv8(cache, torch.zeros(1, 1, dtype=torch.int32),
                              torch.ones(1, dtype=torch.int32), 1, 1, 128)
    with pytest.raises(ValueError):
        kv8.paged_decode_attention_kv8(x[0], cache[:, 0], torch.zeros(5, 1, dtype=torch.int32),
                                       torch.ones(5, dtype=torch.int32), 0.1, 1)
    with pytest.raises(ValueError):
        kv8.varlen_attention_kv8(x[0], cache[:, 0], torch.zeros(1, 1, dtype=torch.int32),
                                 torch.zeros(2, dtype=torch.int32),
                                 torch.ones(1, dtype=torch.int32), 1, 1, 0.1)

"""Softmax weights far below the largest one, in fp16: one key with a small V
dominates by 17.6 nats (weights of 2^-25.4 beside its 1) and thousands of others
hold the output.

The bars, per element, for weights w_j = exp(s_j - max s), S = sum w and A = sum
w |v| / S: the output's rounding, 2^-11 |o| + 2^-25; 2^-11 A for a weight rounded
to 11 bits (the attentions of several queries; the decode attentions hold 22);
2^-11 A for the fp32 arithmetic (40001 terms are 2500 additions of 2^-24 each,
and a score's 128 products as much); 2^-32 sum |v| / S for weights among fp16's
subnormals, when the largest weight is held at 2^7 or above and a subnormal is
off by 2^-25 at most."""
import numpy as np
import pytest
import torch

from aegaeon_amd import attention as A
from aegaeon_amd import kv4
from oracle import kv4_oracle as k4

pytestmark = pytest.mark.gpu

SCALE = 17.6 / 36.0


def _rows(rng, n, D, sink):
    """K, V [n, D] of one kv head: key `sink` holds 6 in dim 0, the others
    noise; V is 1e-3 there and 64 elsewhere, with noise."""
    k = 0.05 * rng.standard_normal((n, D))
    k[:, 0] = 0.0
    k[sink] = 0.0
    k[sink, 0] = 6.0
    v = 64.0 + 4.0 * rng.standard_normal((n, D))
    v[sink] = 1e-3 * rng.standard_normal(D)
    return k.astype(np.float16), v.astype(np.float16)


def _queries(rng, m, Hq, D):
    q = 0.5 * rng.standard_normal((m, Hq, D))
    q[:, :, 0] = 6.0
    return q.astype(np.float16)


def _check(out, q, k, v, limits, weight_bits):
    """out [m, Hq, D] against the definition over k, v [n, D]: query i attends
    to keys j < limits[i]."""
    got, q, k, v = out.double().cpu().numpy(), *(x.astype(np.float64) for x in (q, k, v))
    assert np.isfinite(got).all()
    for i, lim in enumerate(limits):
        s = q[i] @ k[:lim].T * SCALE
        w = np.exp(s - s.max(-1, keepdims=True))
        total = w.sum(-1, keepdims=True)
        want, a = w @ v[:lim] / total, w @ np.abs(v[:lim]) / total
        bar = (2.0 ** -11 * np.abs(want) + 2.0 ** -25
               + (2.0 ** -weight_bits + 2.0 ** -11) * a
               + 2.0 ** -32 * np.abs(v[:lim]).sum(0) / total)
        worst = (np.abs(got[i] - want) / bar).max()
        assert worst <= 1.0, (i, worst, (np.abs(got[i] - want) / np.abs(want)).max())


def _cache4(rng, device, n, D, sink):
    """A 4-bit cache of one sequence and kv head, and the rows it stands for."""
    k, v = _rows(rng, n, D, sink)
    blocks = -(-n // 16)
    table = rng.permutation(blocks)
    slots = torch.from_numpy(table[np.arange(n) // 16] * 16 + np.arange(n) % 16).to(device)
    cache = kv4.kv4_cache(blocks, 1, 1, D, device)
    kv4.reshape_and_cache_kv4(*(torch.from_numpy(x).to(device).unsqueeze(1) for x in (k, v)),
                              cache[:, 0], slots)
    bt = torch.from_numpy(table[None].astype(np.int32)).to(device)
    sl = torch.tensor([n], dtype=torch.int32, device=device)
    return cache[:, 0], bt, sl, *(k4.decode(*k4.encode(x.astype(np.float64), "fp16"))
                                  for x in (k, v))


@pytest.mark.parametrize("m,Hq,D,n", [(1, 4, 128, 40001),   # two key tiles per step
                                      (5, 8, 64, 40001),
                                      (40, 4, 64, 20001),   # four waves
                                      (100, 32, 128, 41001)])  # eight waves
@pytest.mark.parametrize("late", [False, True])
def test_several_queries_over_the_4_bit_cache(device, m, Hq, D, n, late):
    rng = np.random.default_rng(m + D)
    sink = n - 2 * m if late else 3
    cache, bt, sl, k, v = _cache4(rng, device, n, D, sink)
    q = _queries(rng, m, Hq, D)
    cu = torch.tensor([0, m], dtype=torch.int32, device=device)
    out = kv4.varlen_attention_kv4(torch.from_numpy(q).to(device), cache, bt, cu, sl, m, n, SCALE)
    _check(out, q, k, v, n - m + 1 + np.arange(m), 11)


@pytest.mark.parametrize("n,batch,Hq,D", [(700, 3, 8, 64), (700, 3, 4, 128), (4500, 1, 16, 128),
                                          (4500, 1, 8, 64)])
def test_prompts(device, n, batch, Hq, D):
    rng = np.random.default_rng(n + D)
    k, v = _rows(rng, n, D, 3)
    q = _queries(rng, n, Hq, D)
    cu = torch.arange(batch + 1, dtype=torch.int32, device=device) * n
    x = [torch.from_numpy(a.reshape(n, -1, D)).to(device).repeat(batch, 1, 1) for a in (q, k, v)]
    out = A.varlen_prefill_attention(*x, cu, n, SCALE).unflatten(0, (batch, n))
    rows = np.unique(np.concatenate([[0, 2, 3, 4, 63, 64, 65, n - 1], rng.integers(0, n, 40)]))
    for b in range(batch):
        _check(out[b, torch.from_numpy(rows).to(device)], q[rows], k, v, rows + 1, 11)


@pytest.mark.parametrize("Hq,D", [(4, 64), (7, 128), (16, 128), (2, 256)])
@pytest.mark.parametrize("nwg", [0, 1])
def test_decode_over_the_4_bit_cache(device, Hq, D, nwg):
    rng = np.random.default_rng(Hq + D)
    n = 40001
    cache, bt, sl, k, v = _cache4(rng, device, n, D, 3)
    q = _queries(rng, 1, Hq, D)
    out = kv4.paged_decode_attention_kv4(torch.from_numpy(q).to(device), cache, bt, sl, SCALE, n,
                                         n_workgroups=nwg)
    _check(out, q, k, v, [n], 22)


@pytest.mark.parametrize("Hq,D", [(4, 64), (7, 128), (2, 256)])
@pytest.mark.parametrize("nwg", [0, 1])
@pytest.mark.parametrize("appending", [False, True])
def test_decode(device, Hq, D, nwg, appending):
    rng = np.random.default_rng(Hq + D)
    n = 40001
    k, v = _rows(rng, n, D, 3)
    q = _queries(rng, 1, Hq, D)
    blocks = -(-n // 16)
    caches = torch.zeros(2, blocks * 16, 1, D, dtype=torch.float16, device=device)
    held = n - 1 if appending else n
    for c, x in zip(caches, (k, v)):
        c[:held, 0] = torch.from_numpy(x[:held]).to(device)
    new = {}
    if appending:
        new = {name: torch.from_numpy(x[-1].reshape(1, 1, D)).to(device)
               for name, x in (("key", k), ("value", v))}
    kc, vc = caches.view(2, blocks, 16, 1, D)
    bt = torch.arange(blocks, dtype=torch.int32, device=device)[None]
    sl = torch.tensor([n], dtype=torch.int32, device=device)
    out = A.paged_decode_attention(torch.from_numpy(q).to(device), kc, vc, bt, sl, SCALE, n,
                                   n_workgroups=nwg, **new)
    _check(out, q, k, v, [n], 22)

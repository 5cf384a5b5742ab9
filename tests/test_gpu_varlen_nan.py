"""NaN in V of long sequences, attention of several query tokens over the 4- and the
8-bit cache: it shows in its dims of the rows that see its token and in no others,
which keep the bits they have with zeros in its place.  Sequences of more blocks than
a workgroup looks through at once, NaN in the first of them, the last, and between."""
import numpy as np
import pytest
import torch

from aegaeon_amd import kv4, kv8

pytestmark = pytest.mark.gpu


def _cache(bits, blocks, Hkv, D, device):
    if bits == 4:
        return kv4.kv4_cache(blocks, 1, Hkv, D, device=device)[:, 0]
    return kv8.kv8_cache(blocks, 1, Hkv, D, device=device)[:, 0]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,lens,Hq,Hkv,D", [
    ([5] * 40, [5000] + [20] * 39, 64, 64, 64),     # two key tiles a step, whole sequences
    ([70] * 40, [9000] + [80] * 39, 64, 64, 64),    # one
    ([40], [9000], 28, 4, 128),                     # one, cut
    ([3], [30000], 6, 2, 128),                      # two, cut
    ([300], [9000], 80, 40, 128),                   # eight waves
    ([300], [13000], 80, 80, 128)])                 # eight waves, 160 tiles
def test_nan_of_long_sequences(device, bits, dtype, new, lens, Hq, Hkv, D):
    g = torch.Generator(device=device).manual_seed(sum(lens) + D)
    n, m, T = lens[0], new[0], sum(lens)
    rows = [torch.randn(T, Hkv, D, generator=g, device=device).to(dtype) for _ in range(2)]
    width = -(-n // 16)
    tables = torch.zeros(len(lens), width, dtype=torch.int32, device=device)
    slots, at = [], 0
    ids = torch.randperm(sum(-(-x // 16) for x in lens), generator=g, device=device).int()
    for b, x in enumerate(lens):
        k = -(-x // 16)
        tables[b, :k] = ids[at:at + k]
        at += k
        slots.append((tables[b, :k].long()[:, None] * 16
                      + torch.arange(16, device=device)).reshape(-1)[:x])
    slots = torch.cat(slots)
    # of the first sequence: (token, kv head, dim); the last query alone sees the last token
    spots = [(0, 0, 3), (n // 2, Hkv - 1, 7), (n // 2 + 1, Hkv - 1, 7), (n - m, Hkv // 2, 40),
             (n - 1, 1, 63), (16 * 257 + 5, 0, D - 1), (n - 2, 0, D - 1)]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=device)
    sl = torch.tensor(lens, dtype=torch.int32, device=device)
    q = torch.randn(sum(new), Hq, D, generator=g, device=device).to(dtype)
    group = 32 if bits == 4 else 1
    outs = []
    for value in (0.0, float("nan")):
        for t, h, d in spots:
            rows[1][t, h, d // group * group:(d // group + 1) * group] = value
        cache = _cache(bits, ids.numel(), Hkv, D, device)
        put, attend = ((kv4.reshape_and_cache_kv4, kv4.varlen_attention_kv4) if bits == 4 else
                       (kv8.reshape_and_cache_kv8, kv8.varlen_attention_kv8))
        put(rows[0], rows[1], cache, slots)
        outs.append(attend(q, cache, tables, cu, sl, m, n, D ** -0.5))
    nan = torch.zeros(outs[0].shape, dtype=torch.bool, device=device)
    for t, h, d in spots:
        heads = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
        nan[max(t - (n - m), 0):m, heads, d // group * group:(d // group + 1) * group] = True
    assert torch.equal(torch.isnan(outs[1]), nan)
    assert not torch.isnan(outs[0]).any()
    assert torch.equal(outs[1][~nan], outs[0][~nan])

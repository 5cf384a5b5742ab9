"""Forms of the 4-bit cache's attentions that a rule picks by sizes or heads:
the decode kernel's column packing at every head_dim, NaN in V under it, and of
several queries the eight-wave kernel with many pieces per tile, under capture
and on other streams, and pools past 4 GiB.  Bars are those of test_gpu_kv4.py and
test_gpu_kv4_varlen.py."""
import math

import numpy as np
import pytest
import torch

from aegaeon_amd import attention as A
from aegaeon_amd import kv4
from oracle import kv4_oracle as k4
from oracle import kv_oracle as ko
from tests.kvtest_utils import random_bits, to_device_bits
from tests.test_gpu_kv4 import _check_decode, _decode_setup
from tests.test_gpu_kv4_varlen import Batch, within

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

# (query heads, kv heads, head_dim): groups of up to 4, 5 to 8, and 9 to 16 at
# each head_dim
FORMS = [(8, 2, 64), (8, 1, 64), (14, 2, 64), (32, 2, 64), (12, 4, 128), (10, 2, 128),
         (16, 1, 128), (36, 4, 128), (4, 1, 256), (8, 1, 256), (15, 3, 256), (22, 2, 256)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,D", FORMS)
@pytest.mark.parametrize("nwg", [0, 1, 5])
def test_decode_of_every_group_and_head_dim(device, dtype, Hq, Hkv, D, nwg):
    lens = [1, 16, 31, 0, 65, 200, 777, 129]
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, lens, Hq, Hkv, D, dtype,
                                                               Hq * 7 + D + nwg)
    out = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 1 / math.sqrt(D), 777, n_workgroups=nwg)
    assert not out[3].any()
    _check_decode(out, q, cache, tables, lens, 1 / math.sqrt(D), D, dtype)


@pytest.mark.parametrize("batch", [3, 150])
@pytest.mark.parametrize("Hq,Hkv,D", FORMS)
def test_a_plan_gives_the_same_bits(device, batch, Hq, Hkv, D):
    lens = np.random.default_rng(batch + D).integers(0, 150, size=batch)
    lens[0] = 333
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, lens, Hq, Hkv, D, "bf16", 5)
    plain = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 0.1, 333)
    plan = A.DecodePlan(bt, sl, 333, Hkv)
    planned = kv4.paged_decode_attention_kv4(dq, dc, None, None, 0.1, 333, plan=plan)
    assert torch.equal(plain.view(torch.int16), planned.view(torch.int16))
    _check_decode(planned, q, cache, tables, lens, 0.1, D, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,Hkv,D", FORMS)
@pytest.mark.parametrize("token", [0, 37, 49])
def test_decode_a_nan_of_v_shows_in_its_groups_dims_only(device, dtype, Hq, Hkv, D, token):
    rng, lens, tables, cache, q, dc, dq, bt, sl = _decode_setup(device, [50, 20], Hq, Hkv, D, dtype,
                                                               30)
    clean = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 0.1, 50)
    head, grp = Hkv - 1, D // 32 - 1
    dc[tables[0][token // 16], head, 1, 8 * D + grp * 16 + token % 16] = 255
    out = kv4.paged_decode_attention_kv4(dq, dc, bt, sl, 0.1, 50)
    hit = torch.zeros(out.shape, dtype=torch.bool, device=device)
    hit[0, head * (Hq // Hkv):, 32 * grp:32 * grp + 32] = True
    assert torch.isnan(out[hit].float()).all()
    assert torch.equal(out[~hit].view(torch.int16), clean[~hit].view(torch.int16))


@pytest.mark.parametrize("dtype,causal", [("bf16", True), ("bf16", False), ("fp16", True)])
@pytest.mark.parametrize("new,lens", [([100], [41001]), ([90, 5], [41500, 500])])
def test_eight_waves_over_many_pieces(device, dtype, causal, new, lens):
    """Few tiles of very many keys: sixteen pieces a tile and more, four rows to
    a merge workgroup."""
    Hq, Hkv, D = 32, 1, 128
    b = Batch(device, new, lens, Hq, Hkv, D, dtype, new[0])
    # the workspace of eight 32-row units a piece, sixteen pieces a tile and more
    ws = kv4.varlen_attention_workspace(len(new), sum(new), max(new), max(lens), Hq, Hkv, D,
                                        DTYPES[dtype])
    cus = torch.cuda.get_device_properties(device).multi_processor_count
    jobs = min(len(new) * -(-max(new) * Hq // 256), sum(new) * Hq // 256 + len(new))
    assert cus - jobs * 7 // 8 >= 16 * jobs
    assert ws.numel() == (cus - jobs * 7 // 8 + jobs) * 256 * (D * 4 + 8) + 256 + 24 * jobs
    out = b.run(0.09, causal)
    b.check(out, 0.09, causal)
    assert torch.equal(out.view(torch.int16), b.run(0.09, causal).view(torch.int16))


def test_eight_waves_captured(device):
    """Captured on one stream, replayed with eager calls of other sizes between
    and new inputs: every replay equals the eager result."""
    b = Batch(device, [600], [6001], 40, 2, 128, "bf16", 3)
    other = Batch(device, [64], [20000], 14, 2, 128, "bf16", 4)
    out = torch.empty_like(b.dq)
    b.run(0.1)
    other.run(0.1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        b.run(0.1, out=out)
    for _ in range(4):
        b.dq.mul_(-1.25)
        want = b.run(0.1)
        other.run(0.1)
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("new,lens,Hq,Hkv,D", [([5, 40], [3000, 700], 28, 4, 128),
                                               ([600], [6001], 40, 2, 128),
                                               ([100], [41001], 32, 1, 128)])
def test_several_queries_on_another_stream(device, new, lens, Hq, Hkv, D):
    b = Batch(device, new, lens, Hq, Hkv, D, "fp16", 6)
    want = b.run(0.1)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = [b.run(0.1) for _ in range(3)]
    again = b.run(0.1)  # beside the other stream's
    torch.cuda.synchronize()
    for x in got + [again]:
        assert torch.equal(x.view(torch.int16), want.view(torch.int16))
    b.check(want, 0.1)


@pytest.mark.parametrize("m,Hq", [(3, 4), (30, 4), (70, 40)])
def test_several_queries_in_a_pool_past_32_bit_offsets(device, m, Hq):
    """Blocks whose byte offset passes 2^32, under each kernel (the last: eight
    waves, by the host's bound of the keys)."""
    D, n, layers = 128, 70000, 32  # 69632 bytes per block, 4.87e9 in all
    cache = torch.empty((n, layers, 1, 2, 1088), dtype=torch.uint8, device=device)
    rng = np.random.default_rng(m)
    longest = 40 * 16
    table = [n - 1 - 3 * i for i in range(20)] + [5 + 7 * i for i in range(20)]
    x = random_bits(rng, (2, longest, 1, D), "bf16")
    slots = np.array([table[i // 16] * 16 + i % 16 for i in range(longest)])
    dx = to_device_bits(x, "bf16", device)
    kv4.reshape_and_cache_kv4(dx[0], dx[1], cache[:, 31], torch.from_numpy(slots).to(device))
    bound = 80000
    bt = torch.zeros(1, bound // 16, dtype=torch.int32, device=device)
    bt[0, :40] = torch.tensor(table, dtype=torch.int32)
    q = random_bits(rng, (m, Hq, D), "bf16")
    cu = torch.tensor([0, m], dtype=torch.int32, device=device)
    sl = torch.tensor([longest], dtype=torch.int32, device=device)
    out = kv4.varlen_attention_kv4(to_device_bits(q, "bf16", device), cache[:, 31], bt, cu, sl, m,
                                   bound, 0.1)
    rows = [k4.decode(*k4.encode(ko.bits_to_float(a, "bf16"), "bf16")).reshape(40, 16, 1, D)
            for a in x]
    want = k4.varlen_attention(ko.bits_to_float(q, "bf16"), *rows, [list(range(40))], [0, m],
                               [longest], 0.1, True)
    within(out.double().cpu().numpy(), want, "bf16")

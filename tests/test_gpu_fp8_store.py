"""store_kvcache_fp8 on the GPU: codes and scales bit for bit against the oracle."""
import pytest
import torch

from fp8_cases import planes_on, random_planes, to_codes
from nano_vllm_b200 import _lib, attention as A
from oracle import fp8_cache_ref as F8

pytestmark = pytest.mark.gpu


def check(cuda, key, value, planes, slots, status=0, repeat=1):
    """One call against the oracle; returns the planes afterwards, on the CPU."""
    dev = planes_on(cuda, *planes)
    _lib.read_status()
    for _ in range(repeat):
        A.store_kvcache_fp8(key.to(cuda), value.to(cuda), *dev, slots.to(cuda))
    torch.cuda.synchronize()
    assert _lib.read_status() == status
    ref = [t.clone() for t in planes]
    F8.store_kvcache_fp8_ref(key, value, *ref, slots)
    got = [to_codes(dev[0]), to_codes(dev[1]), dev[2].cpu(), dev[3].cpu()]
    for what, a, b in zip(("k codes", "v codes", "k scales", "v scales"), got, ref):
        same = (a == b) | (a.isnan() & b.isnan() if a.is_floating_point() else False)
        assert same.all(), f"{what}: {int((~same).sum())} differ, first at {(~same).nonzero()[0].tolist()}"
    return got


def rows(gen, n, hkv, d, spread=1.0):
    return (torch.randn(n, hkv, d, generator=gen) * torch.exp(spread * torch.randn(n, hkv, 1, generator=gen))).bfloat16()


def prompt_slots(gen, lens, blocks):
    """Slots of whole sequences, one after the other, in random blocks; (start, tokens) of each."""
    order, out, at = torch.randperm(blocks, generator=gen).tolist(), [], 0
    for start, n in lens:
        need = -(-(start + n) // 256)
        ids = order[at:at + need]
        at += need
        out += [ids[p // 256] * 256 + p % 256 for p in range(start, start + n)]
    return torch.tensor(out, dtype=torch.int32)


@pytest.mark.parametrize("hkv,d", [(8, 128), (2, 64), (1, 128), (1, 64), (3, 128), (11, 64)])
@pytest.mark.parametrize("lens", [[(0, 1)], [(5, 1)], [(15, 2)], [(0, 16)], [(0, 17)], [(7, 40)], [(0, 300), (255, 3), (16, 1), (30, 100)]])
def test_sequences(cuda, hkv, d, lens):
    g = torch.Generator().manual_seed(hkv * 1000 + d + len(lens))
    slots = prompt_slots(g, lens, 8)
    check(cuda, rows(g, len(slots), hkv, d), rows(g, len(slots), hkv, d), random_planes(g, 8, hkv, d), slots)


@pytest.mark.parametrize("hkv,d", [(2, 128), (2, 64)])
@pytest.mark.parametrize("n", [4096, 4097, 4117])
def test_many_rows(cuda, hkv, d, n):
    """One row to a thread block, then sixteen: groups that lie across blocks."""
    g = torch.Generator().manual_seed(n)
    lens = [(3, 1000), (0, 900), (250, 21), (17, 2100)]
    lens.append((9, n - sum(m for _, m in lens)))
    slots = prompt_slots(g, lens, 22)
    check(cuda, rows(g, n, hkv, d), rows(g, n, hkv, d), random_planes(g, 22, hkv, d), slots)


@pytest.mark.parametrize("hkv,d", [(8, 128), (2, 64)])
def test_decode_rows_grow_their_groups(cuda, hkv, d):
    """One row per sequence at every offset, a fifth of them far larger than what is there, some rows skipped."""
    g = torch.Generator().manual_seed(7)
    n = 64
    blocks = torch.randperm(n, generator=g).to(torch.int32)
    slots = blocks * 256 + 16 * (torch.arange(n, dtype=torch.int32) % 5) + torch.arange(n, dtype=torch.int32) % 16
    slots[::9] = -1
    size = torch.where(torch.arange(n) % 5 == 0, 300.0, 1.0).view(n, 1, 1)
    key, value = rows(g, n, hkv, d), rows(g, n, hkv, d)
    key, value = (key.float() * size).bfloat16(), (value.float() * size.flip(0)).bfloat16()
    planes = random_planes(g, n, hkv, d, spread=0.3)
    once = check(cuda, key, value, planes, slots)
    twice = check(cuda, key, value, planes, slots, repeat=2)  # the same rows again change nothing
    assert all(torch.equal(a, b) for a, b in zip(once, twice))


def test_rows_skipped_between_rows_of_a_group(cuda):
    g = torch.Generator().manual_seed(8)
    slots = torch.full((150,), -1, dtype=torch.int32)
    slots[3], slots[50], slots[51], slots[120] = 256 + 16, 256 + 17, 256 + 18, 256 + 19  # one group, gaps wider than a warp
    slots[121], slots[149] = 256 + 32, 256 + 33
    for hkv, d in ((2, 128), (3, 64)):
        check(cuda, rows(g, 150, hkv, d), rows(g, 150, hkv, d), random_planes(g, 3, hkv, d), slots)


@pytest.mark.parametrize("hkv,d", [(2, 128), (3, 64)])
@pytest.mark.parametrize("n", [2, 16, 17, 33, 100])
def test_the_same_slot_again_and_again(cuda, hkv, d, n):
    """The last row stays, as a list of stores would leave it."""
    g = torch.Generator().manual_seed(n)
    planes = random_planes(g, 2, hkv, d)
    check(cuda, rows(g, n, hkv, d), rows(g, n, hkv, d), planes, torch.zeros(n, dtype=torch.int32))
    pairs = torch.arange(n, dtype=torch.int32) // 3 % 16 + 32
    check(cuda, rows(g, n, hkv, d), rows(g, n, hkv, d), planes, pairs.sort().values)


def test_values_that_are_hard(cuda):
    """Nothing, negative zero, ties, the borders of a scale, subnormal and huge numbers, NaN and infinities."""
    g = torch.Generator().manual_seed(9)
    hkv, d = 2, 128
    key, value = rows(g, 200, hkv, d), rows(g, 200, hkv, d)
    key[0:16] = 0.0
    key[16] = -0.0
    key[32, 0, :5] = torch.tensor([448.0, 1.0, 1.0625, 1.1875, -1.0625])
    key[48, 0], key[64, 0] = 448.0, 450.0
    key[80, 1], key[96, 1], key[112, 1] = 3e38, 1e-30, 1e-39
    value[5, 0, 3], value[20, 1, 7], value[40, 0, 9] = float("nan"), float("inf"), float("-inf")
    value[160:176] = float("nan")
    value[177:180] = float("inf")
    slots = torch.arange(200, dtype=torch.int32)
    check(cuda, key, value, random_planes(g, 1, hkv, d), slots)
    check(cuda, value, key, random_planes(g, 1, hkv, d), slots + 8)


def test_scales_that_no_store_wrote(cuda):
    """Rows appended to groups whose scale is zero, no power of two, tiny, huge."""
    g = torch.Generator().manual_seed(10)
    hkv, d = 8, 128
    planes = random_planes(g, 1, hkv, d)
    for s in planes[2:]:
        s[0, :, 0] = torch.tensor([0.0, 0.3, 1e-30, 5e-39, 1.5, 0.75, 3.0, 7e20])
    check(cuda, rows(g, 1, hkv, d), rows(g, 1, hkv, d), planes, torch.tensor([9], dtype=torch.int32))


def test_strided_rows_and_slots_outside_the_cache(cuda):
    g = torch.Generator().manual_seed(11)
    n, hq, hkv, d = 90, 4, 2, 64
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g).bfloat16()
    _, k, v = qkv.split([hq * d, hkv * d, hkv * d], dim=-1)
    slots = prompt_slots(g, [(0, 90)], 3)
    slots[4] = 3 * 256
    slots[70] = 2 ** 31 - 1
    check(cuda, k.view(n, hkv, d), v.view(n, hkv, d), random_planes(g, 3, hkv, d), slots, status=1)


def test_no_rows_and_other_streams(cuda):
    g = torch.Generator().manual_seed(12)
    planes = random_planes(g, 2, 2, 64)
    check(cuda, rows(g, 0, 2, 64), rows(g, 0, 2, 64), planes, torch.zeros(0, dtype=torch.int32))
    key, value, slots = rows(g, 40, 2, 64).to(cuda), rows(g, 40, 2, 64).to(cuda), torch.arange(40, dtype=torch.int32, device=cuda)
    here, there = planes_on(cuda, *planes), planes_on(cuda, *planes)
    A.store_kvcache_fp8(key, value, *here, slots)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        A.store_kvcache_fp8(key, value, *there, slots)
    stream.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(here, there))

"""Attention over the cache where weights are far apart: a dominant key and what thousands of others add to it."""
import pytest
import torch

import frisk_b200 as F
from oracle import cache_oracle as co
from tests.test_cache_gpu import Batch, attend

pytestmark = pytest.mark.gpu


def with_a_sink(counts, lengths, hkv, group, d, dtype, held, nats, at=0, apart=0):
    """A batch whose key ``at`` of every sequence scores ``nats`` above the others, its value 0.01 beside theirs about 1.  ``apart``: every
    64th key scores 280 / sqrt(D) below the others, and its values' scale (8-bit) is 2^apart times theirs."""
    b = Batch(counts, lengths, hkv, group, d, 64, dtype, held, 21)
    g = torch.Generator().manual_seed(5)
    size = 40.0 if apart else 4.0
    b.q[:, :, 0] = size
    cpu = [t.clone() for t in b.cpu]
    for n, (count, length) in enumerate(zip(counts, lengths)):
        j = torch.arange(count + length)
        where = b.table_cpu[n].long()[j // 64], slice(None), j % 64
        k, v = 0.05 * torch.randn(len(j), hkv, d, generator=g), 1.0 + 0.1 * torch.randn(len(j), hkv, d, generator=g)
        k[:, :, 0] = 0.0
        k[at], v[at] = 0.0, 0.01
        k[at, :, 0] = nats * d ** 0.5 / size
        if apart:
            k[5::64] = 0.0
            k[5::64, :, 0] = -7.0
        for i, x in enumerate((k, v)):
            if len(cpu) == 4:  # 2^-6: keys up to 7, 2^-8: values up to 1.75
                cpu[i][where] = (x * 2.0 ** (6 + 2 * i)).to(torch.float8_e4m3fn)
                cpu[2 + i][where] = 127 - 6 - 2 * i
                if apart and i:
                    cpu[3][b.table_cpu[n].long()[j[5::64] // 64], :, j[5::64] % 64] += apart
            else:
                cpu[i][where] = x.to(dtype)
    if len(cpu) == 4:  # larger keys: another scale
        for n in range(len(counts)):
            where = int(b.table_cpu[n, at // 64]), slice(None), at % 64
            cpu[0][where] = torch.zeros(hkv, d).to(torch.float8_e4m3fn)
            cpu[0][where[0], :, where[2], 0] = torch.tensor(nats * d ** 0.5 / size * 8.0).to(torch.float8_e4m3fn)
            cpu[2][where] = 124
    b.cpu = tuple(cpu)
    b.refresh()
    return b


# (one head's parts shared by many CTAs; several whole items a CTA; more rows than a tile)
SINKS = [([5], [32000], 1, 8, 64), ([3] * 40, [200 + 9 * i for i in range(40)], 8, 2, 128), ([70], [4000], 1, 4, 128)]


@pytest.mark.parametrize("nats", [6.0, 8.0, 10.0, 11.0, 14.0])
@pytest.mark.parametrize("counts,lengths,hkv,group,d", SINKS)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("held", [None, "float8_e4m3fn"])
def test_the_others_beside_a_dominant_key(nats, counts, lengths, hkv, group, d, dtype, held):
    """What the others weigh is in the results of every kernel, however the choice among them falls."""
    b = with_a_sink(counts, lengths, hkv, group, d, getattr(torch, dtype), held and getattr(torch, held), nats)
    for rows in (16, 128, 256):
        attend(b, tile_rows=rows)
    for hint in (1, 64):
        attend(b, tile_rows=0, max_new=hint)


@pytest.mark.parametrize("nats", [6.0, 12.0, 14.0, 15.5])
@pytest.mark.parametrize("apart", [4, 5, 8])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_scales_that_no_weight_stands_behind(nats, apart, dtype):
    """Keys that weigh little and have larger values' scales than the others, one in every tile."""
    b = with_a_sink([6] * 20, [1900 + 17 * i for i in range(20)], 2, 3, 64, getattr(torch, dtype), torch.float8_e4m3fn, nats, apart=apart)
    for rows in (16, 128, 256):
        attend(b, tile_rows=rows)


@pytest.mark.parametrize("first,then", [(243, 80), (67, 187), (243, 107), (230, 66)])
@pytest.mark.parametrize("count,length", [(40, 700), (130, 128), (70, 64)])
def test_values_of_tiles_far_apart(first, then, count, length):
    """Values' scales of the first 64 keys, near the end of the type's range, and of the others: the row sum keeps its range."""
    counts, lengths = [count] + [3] * 60, [length] + [500 + 7 * i for i in range(60)]  # (a CTA has whole items)
    b = Batch(counts, lengths, 4, 1, 64, 64, torch.bfloat16, torch.float8_e4m3fn, 22)
    g = torch.Generator().manual_seed(3)
    cpu = [t.clone() for t in b.cpu]
    for n, keys in enumerate(x + y for x, y in zip(counts, lengths)):
        j = torch.arange(keys)
        where = b.table_cpu[n].long()[j // 64], slice(None), j % 64
        cpu[1][where] = (2.0 * torch.randn(keys, 4, 64, generator=g)).clamp(-4, 4).to(torch.float8_e4m3fn)
        cpu[2][where] = 117
        cpu[3][where] = torch.where(j < 64, first, then).to(torch.uint8)[:, None]
    b.cpu = tuple(cpu)
    b.refresh()
    alone = torch.eye(count, dtype=torch.bool)  # whole tiles of new tokens that a row does not see
    alone = torch.cat([alone] + [alone[:3]] * 60)
    for rows in (16, 128, 256):
        attend(b, tile_rows=rows)
        attend(b, tile_rows=rows, mask=alone)


@pytest.mark.parametrize("nats", [17.3, 18.0])
@pytest.mark.parametrize("dtype,held", [("float16", None), ("bfloat16", None), ("float16", "float8_e4m3fn"), ("bfloat16", "float8_e4m3fn")])
def test_sixty_thousand_keys_beside_a_dominant_one(nats, dtype, held):
    """160 sequences over the same pages, so that a CTA holds all keys of one."""
    many, length = 160, 59_999
    b = with_a_sink([1], [length], 1, 8, 64, getattr(torch, dtype), held and getattr(torch, held), nats)
    q, plan = b.q.expand(many, -1, -1).contiguous(), [b.plan[0].expand(many, -1).contiguous()]
    plan += [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (range(many + 1), [length] * many)]
    for rows in (16, 128, 256):
        out = F.cache_attention(b.cache, q, *plan, tile_rows=rows).cpu().double()
        F.cache_check()
        ref, bound = co.attention(b.cpu, b.q.cpu(), *b.host, terms=held is not None and rows > 16)
        assert bool(((out - ref).abs() <= bound).all()), (rows, float((out - ref).abs().max()), float(bound.max()))


@pytest.mark.parametrize("held", [None, "float8_e4m3fn"])
@pytest.mark.parametrize("counts,lengths,hkv", [([5, 1], [700, 64], 2), ([3] * 40, [600 + i for i in range(40)], 4), ([200], [9000], 1)])
def test_sums_of_values_near_the_end_of_the_range_are_finite(held, counts, lengths, hkv):
    b = Batch(counts, lengths, hkv, 2, 64, 64, torch.bfloat16, held and getattr(torch, held), 23)
    cpu = [t.clone() for t in b.cpu]
    sign = torch.where(torch.arange(64) % 3 == 0, -1.0, 1.0)
    for n, keys in enumerate(x + y for x, y in zip(counts, lengths)):
        j = torch.arange(keys)
        where = b.table_cpu[n].long()[j // 64], slice(None), j % 64
        if held:  # 240 * 2^120 is 0.94 of the largest bf16 value
            cpu[1][where] = (240.0 * sign).expand(keys, hkv, 64).to(torch.float8_e4m3fn)
            cpu[2][where], cpu[3][where] = 117, 247
        else:
            cpu[1][where] = (3.2e38 * sign).expand(keys, hkv, 64).to(torch.bfloat16)
            cpu[0][where] = (0.1 * cpu[0][where].float()).to(torch.bfloat16)
    b.cpu = tuple(cpu)
    b.refresh()
    for rows in (16, 128, 256):
        assert bool((attend(b, tile_rows=rows)[b.inside()].abs() > 3e38).all())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_the_largest_values_stay_finite(dtype):
    """All values are the largest of the type, and a late key outweighs the others by less than moves the reference: its weight is rounded,
    in some rows up."""
    dtype = getattr(torch, dtype)
    b = Batch([1] * 20, [64 * 3 + i for i in range(20)], 1, 16, 64, 64, dtype, None, 24)
    cpu = [t.clone() for t in b.cpu]
    for n, length in enumerate(b.lengths):
        j = torch.arange(length + 1)
        where = b.table_cpu[n].long()[j // 64], slice(None), j % 64
        cpu[1][where] = torch.where(torch.arange(64) % 2 == 0, -1.0, 1.0).to(dtype) * torch.finfo(dtype).max
        cpu[0][where] = 0.0
        cpu[0][where[0], :, where[2], 1] = -30.0
        cpu[0][int(b.table_cpu[n, 0]), :, 0, 1] = 0.0
        cpu[0][int(b.table_cpu[n, 2]), :, 11, 0] = 1.0
        cpu[0][int(b.table_cpu[n, 2]), :, 11, 1] = 0.0
    b.cpu = tuple(cpu)
    b.refresh()
    b.q[:, :, 1] = 16.0  # one key at 0, one late key, the others far below
    b.q[:, :, 0] = 16 + (torch.arange(20 * 16, device="cuda").view(20, 16) / 16).to(dtype)  # 2 to 4.5 above: 2^2.9 to 2^6.5
    for rows in (16, 128, 256):
        assert bool((attend(b, tile_rows=rows).abs() > 0.98 * torch.finfo(dtype).max).all())

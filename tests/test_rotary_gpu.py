"""Rotary positions and their gradients against 64 bits.

Bound for one result a c - b s: half a step of its type, and in 32 bits the argument of sine and cosine (2^-24 of at most half a turn:
pi 2^-24 on the angle), sine and cosine themselves (2 units of 2^-24), the amplitude (1), the products and their sum (3): less than
10 x 2^-24 of amplitude (|a| + |b|)."""
import math

import pytest

from oracle import cache_oracle as co

pytestmark = pytest.mark.gpu


def rows(n, h, hkv, d, dtype, seed, device="cuda"):
    """Queries and keys as columns of one buffer, with columns of something else around them."""
    import torch
    g = torch.Generator().manual_seed(seed)
    pitch = (h + 2 * hkv) * d
    buf = torch.randn(n, pitch, generator=g).to(dtype).to(device)
    return buf, buf[:, :h * d].view(n, h, d), buf[:, h * d:(h + hkv) * d].view(n, hkv, d)


def close(got, x, positions, f, amplitude, interleaved, inverse):
    import torch
    x = x.cpu()
    ref = co.rotary(x, positions.cpu(), f.cpu(), amplitude, interleaved, inverse)
    half = len(f)
    size = torch.zeros_like(ref)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        size[..., a] = size[..., b] = x[..., a].double().abs() + x[..., b].double().abs()
    bound = co.H[x.dtype] * ref.abs() * (1 + 1e-6) + 10 * 2.0 ** -24 * amplitude * size
    assert torch.equal(got.cpu()[..., 2 * half:], x[..., 2 * half:])
    off = (got.cpu().double() - ref).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("n,h,hkv,d,dim", [(1, 4, 1, 128, 128), (3, 8, 8, 64, 64), (257, 5, 1, 80, 40), (130, 3, 2, 96, 50), (33, 1, 1, 2, 2),
                                           (700, 16, 4, 128, 64), (5, 2, 1, 7, 6), (9, 2, 2, 256, 256)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary(n, h, hkv, d, dim, dtype, interleaved):
    import torch
    import frisk_b200 as F
    buf, q, k = rows(n, h, hkv, d, getattr(torch, dtype), n + d)
    before = buf.clone()
    positions = torch.arange(n, device="cuda") * 977 + 1_000_003
    f, a = F.rotary_frequencies(dim, scaling="yarn", factor=4.0, trained=4096)
    for inverse, turn in ((False, F.rotary), (True, F.rotary_backward)):
        q2, k2 = turn(q, k, positions, f, amplitude=a, interleaved=interleaved)
        close(q2, q, positions, f, a, interleaved, inverse)
        close(k2, k, positions, f, a, interleaved, inverse)
    q3, none = F.rotary(q, None, positions.int(), f, amplitude=a, interleaved=interleaved)
    assert none is None and torch.equal(q3, F.rotary(q, k, positions, f, amplitude=a, interleaved=interleaved)[0])
    assert torch.equal(buf.view(torch.uint8), before.view(torch.uint8))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,dim", [(128, 128), (80, 40), (10, 6)])
def test_in_place_touches_nothing_else(d, dim, interleaved):
    import torch
    import frisk_b200 as F
    buf, q, k = rows(65, 4, 2, d, torch.bfloat16, 3)
    before = buf.clone()
    positions = torch.randint(-50, 1 << 20, (65,), device="cuda")
    f, _ = F.rotary_frequencies(dim)
    q2, k2 = F.rotary(q.clone(), k.clone(), positions, f, interleaved=interleaved)
    got = F.rotary(q, k, positions, f, interleaved=interleaved, out=(q, k))
    assert got[0] is q and torch.equal(q, q2) and torch.equal(k, k2)
    assert torch.equal(buf[:, 6 * d:], before[:, 6 * d:])


def test_far_positions_and_the_turn_back():
    import torch
    import frisk_b200 as F
    x = torch.randn(64, 2, 64, device="cuda")
    positions = torch.arange(64, device="cuda") * 33_554_393 + 2_000_000_011  # beyond 32 bits
    f, _ = F.rotary_frequencies(64)
    y, _ = F.rotary(x, None, positions, f)
    # 64-bit angles of 4e9 radians: 2^-53 of that for product and reduction each, in the reference too
    ref = co.rotary(x.cpu(), positions.cpu(), f.cpu())
    assert float((y.cpu().double() - ref).abs().max()) < 4 * 4.2e9 * 2.0 ** -52 + 10 * 2.0 ** -24 * 10
    back, _ = F.rotary_backward(y, None, positions, f)
    assert float((back - x).abs().max()) < 25 * 2.0 ** -24 * 10


def test_gradients_against_differences():
    """The map is linear: (f(x + e d) - f(x - e d)) / 2e is f(d), and <f(d), g> = <d, backward(g)>."""
    import torch
    import frisk_b200 as F
    n, h, d = 37, 3, 32
    g = torch.Generator().manual_seed(5)
    x, step, grad = (torch.randn(n, h, d, generator=g).cuda() for _ in range(3))
    positions = torch.arange(n, device="cuda", dtype=torch.int32)
    f, a = F.rotary_frequencies(24, scaling="yarn", factor=8.0, trained=64)
    up, down = (F.rotary(x + s * 0.5 * step, None, positions, f, amplitude=a)[0] for s in (1, -1))
    slope = (up.double() - down.double()).mul(grad.double()).sum().item()
    back, _ = F.rotary_backward(grad, None, positions, f, amplitude=a)
    # n h d terms of size about 2, each 2^-20 off at most
    assert abs(slope - back.double().mul(step.double()).sum().item()) < n * h * d * 8 * 2.0 ** -20


def test_broadcast_gradients_strides_and_empty():
    import torch
    import frisk_b200 as F
    f, _ = F.rotary_frequencies(64)
    positions = torch.arange(40, device="cuda")
    one = torch.randn(1, 1, 64, device="cuda", dtype=torch.float16)
    q, _ = F.rotary(one.expand(40, 6, 64), None, positions, f)  # every stride zero
    assert torch.equal(q, F.rotary(one.expand(40, 6, 64).contiguous(), None, positions, f)[0])
    heads_first = torch.randn(6, 40, 64, device="cuda").transpose(0, 1)
    assert torch.equal(F.rotary(heads_first, None, positions, f)[0], F.rotary(heads_first.contiguous(), None, positions, f)[0])
    odd = torch.randn(40 * 6 * 64 + 1, device="cuda").half()[1:].view(40, 6, 64)  # off 16 bytes
    assert torch.equal(F.rotary(odd, None, positions, f)[0], F.rotary(odd.clone(), None, positions, f)[0])
    e, _ = F.rotary(odd[:0], None, positions[:0], f)
    assert e.shape == (0, 6, 64)


def test_special_values_stay_in_their_pair():
    import torch
    import frisk_b200 as F
    x = torch.ones(4, 1, 16, device="cuda")
    x[1, 0, 3] = math.inf
    x[2, 0, 5] = math.nan
    f, _ = F.rotary_frequencies(16)
    y = F.rotary(x, None, torch.arange(4, device="cuda") + 1, f)[0].cpu()
    bad = ~torch.isfinite(y)
    want = torch.zeros(4, 1, 16, dtype=torch.bool)
    want[1, 0, [3, 11]] = want[2, 0, [5, 13]] = True
    assert torch.equal(bad, want)


def test_captured_and_on_another_stream():
    import torch
    import frisk_b200 as F
    buf, q, k = rows(100, 4, 2, 64, torch.bfloat16, 9)
    f, _ = F.rotary_frequencies(64)
    positions = torch.arange(100, device="cuda")
    want = F.rotary(q, k, positions, f)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = F.rotary(q, k, positions, f, stream=side)
    got2 = F.rotary(q, k, positions, f, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, got2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.rotary(q, k, positions, f)
    positions += 17
    graph.replay()
    want = F.rotary(q, k, positions, f)
    assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_refusals():
    import torch
    import frisk_b200 as F
    buf, q, k = rows(8, 4, 2, 64, torch.float16, 1)
    f, _ = F.rotary_frequencies(64)
    positions = torch.arange(8, device="cuda")
    for bad in (lambda: F.rotary(q.double(), None, positions, f), lambda: F.rotary(q, k.float(), positions, f),
                lambda: F.rotary(q, k, positions[:7], f), lambda: F.rotary(q, k, positions.float(), f), lambda: F.rotary(q, k, positions, f.float()),
                lambda: F.rotary(q.cpu(), None, positions, f), lambda: F.rotary(q, k, positions, torch.cat((f, f))),
                lambda: F.rotary(q, k, positions, f[:0]), lambda: F.rotary(q.transpose(1, 2), None, positions, f),
                lambda: F.rotary(q, k, positions, f, out=(q[1:], k[1:])), lambda: F.rotary(q, k, positions, f, out=(q, q[:, :2])),
                lambda: F.rotary(q, k, positions, f, out=(torch.empty(1, 1, 64, device="cuda", dtype=q.dtype).expand(8, 4, 64), k)),
                lambda: F.rotary(buf[:7, :256].view(7, 4, 64), None, positions[:7], f, out=(buf[1:, :256].view(7, 4, 64), None)),
                lambda: F.rotary(buf[:, :256].view(8, 4, 64), None, positions, f, out=(buf[:, 64:320].view(8, 4, 64), None))):
        with pytest.raises(ValueError):
            bad()
    F.cache_check()

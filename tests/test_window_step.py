"""One new token over the ring of keys and values, and filling the ring.

Would fail if: a slot were read for the wrong position (before, at and past the
ring's first turn), the new row were missed or written elsewhere, a lane's share
of a head width were permuted, splits joined wrongly, an idle sequence touched,
or rows outside the window (NaN planted there) reached the result.
"""

import math

import pytest
import torch

from elysium_wan_b200 import ops


def plain64(qkv, hist, pos, H, hd, Hkv, window, sinks):
    """o in 64 bits from every sequence's whole history of k | v rows."""
    out = torch.zeros(len(pos), H, hd, dtype=torch.float64, device=qkv.device)
    for b, p in enumerate(pos):
        if p < 0:
            continue
        j = torch.arange(p + 1, device=qkv.device)
        j = j[(p - j < window) | (j < sinks)]
        kv = torch.cat([hist[b][:p], qkv[b:b + 1, H * hd:]])[j].double().view(-1, 2, Hkv, hd)
        q = qkv[b, :H * hd].double().view(Hkv, -1, hd)
        w = torch.softmax(q @ kv[:, 0].permute(1, 2, 0) / math.sqrt(hd), -1)
        out[b] = (w @ kv[:, 1].transpose(0, 1)).reshape(H, hd)
    return out.view(len(pos), -1)


def case(pos, H, hd, Hkv, window, sinks, slots, dev, dtype, junk=math.nan, seed=0):
    """qkv, a ring that holds each sequence's history (junk where the token
    may not look), and that history."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    B, width = len(pos), 2 * Hkv * hd
    qkv = torch.randn(B, H * hd + width, generator=g, device=dev).to(dtype)
    hist = [torch.randn(max(p, 0), width, generator=g, device=dev).to(dtype) for p in pos]
    cache = torch.full((B, slots, width), junk, device=dev, dtype=dtype)
    for b, p in enumerate(pos):
        if p <= 0:
            continue
        j = torch.arange(p, device=dev)
        j = j[(p - j < min(window, slots - sinks)) | (j < sinks)]
        cache[b, ops.ring_slot(j, sinks, slots)] = hist[b][j]
    return qkv, cache, hist


def check(pos, H, hd, Hkv, window, sinks, slots, dev, dtype, tol, cache=None):
    qkv, ring, hist = case(pos, H, hd, Hkv, window, sinks, slots, dev, dtype)
    if cache is not None:
        cache.copy_(ring)
        ring = cache
    before = ring.clone()
    t = torch.tensor(pos, device=dev, dtype=torch.int64)
    o = ops.window_attention_step(qkv, ring, t, H, hd, Hkv, window=window, sinks=sinks)
    want = plain64(qkv, hist, pos, H, hd, Hkv, min(window, slots - sinks), sinks)
    for b, p in enumerate(pos):
        if p >= 0:
            before[b, ops.ring_slot(p, sinks, slots)] = qkv[b, H * hd:]
        else:
            assert bool((o[b] == 0).all())
    assert torch.equal(ring.nan_to_num(7.0), before.nan_to_num(7.0))
    assert bool(((o.double() - want).abs() <= tol * (want.abs() + 1.0)).all())
    return qkv, ring, t, o


def test_host_path_and_ring():
    for window, sinks, slots in ((4, 2, 6), (4, 0, 4), (3, 2, 9), (50, 3, 7), (1, 0, 1)):
        pos = [0, 1, 2, 5, 6, 7, 13, 100, -1]
        check(pos, 4, 8, 2, window, sinks, slots, "cpu", torch.float32, 1e-5)
    assert [ops.ring_slot(p, 2, 5) for p in range(9)] == [0, 1, 2, 3, 4, 2, 3, 4, 2]


def test_host_fill_then_step_equals_the_training_rows():
    B, S, H, hd, Hkv, window, sinks = 2, 11, 4, 8, 2, 4, 2
    qkv = torch.randn(B * S, (H + 2 * Hkv) * hd)
    o, _ = ops.window_attention_fwd(qkv, B, S, H, hd, Hkv, window=window, sinks=sinks)
    rows = qkv.view(B, S, -1)
    n = 6
    cache = torch.zeros(B, sinks + window, 2 * Hkv * hd)
    ops.window_cache_fill(rows[:, :n].reshape(B * n, -1), cache, B, n, H, hd, Hkv, sinks=sinks)
    for p in range(n, S):
        got = ops.window_attention_step(rows[:, p].contiguous(), cache, torch.full((B,), p), H, hd, Hkv,
                                        window=window, sinks=sinks)
        assert torch.allclose(got, o.view(B, S, -1)[:, p], atol=1e-5)


def test_refusals_host():
    q, c, p = torch.zeros(2, 64), torch.zeros(2, 4, 32), torch.zeros(2, dtype=torch.int64)
    ops.window_attention_step(q, c, p, 4, 8, 2, window=2)
    for kw in (dict(window=0), dict(window=2, sinks=-1), dict(window=2, sinks=4)):
        with pytest.raises(ValueError):
            ops.window_attention_step(q, c, p, 4, 8, 2, **kw)
    with pytest.raises(ValueError):
        ops.window_attention_step(q, c[:1], p, 4, 8, 2, window=2)
    with pytest.raises(ValueError):
        ops.window_attention_step(q, c, p, 3, 8, 2, window=2)


# ----------------------------------------------------------------------------- GPU
# bf16 output: half a unit, 2^-8 of the value at most; scores and sums are fp32, weights
# keep 16 bits (2^-17 of the values they weigh, all of size about 1 to 4).
TOL = 2.0**-8 * 1.05 + 2.0**-14


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 80, 96, 128])
@pytest.mark.parametrize("H,Hkv", [(4, 4), (4, 2), (12, 1), (40, 2)])
def test_gpu_heads(cuda, hd, H, Hkv):
    pos = [0, 1, 15, 16, 17, 63, 64, 200, 1000, -1, 131]
    check(pos, H, hd, Hkv, 100, 3, 103, cuda, torch.bfloat16, TOL)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks,slots", [(1, 0, 1), (1, 4, 5), (16, 0, 16), (33, 1, 40),
                                                (500, 64, 564), (4000, 4, 2000), (2048, 16, 5000)])
@pytest.mark.parametrize("B", [1, 5, 70])
def test_gpu_windows(cuda, window, sinks, slots, B):
    g = torch.Generator()
    g.manual_seed(B + window)
    pos = [0, sinks, slots - 1, slots, 3 * slots + 1][:max(1, min(5, B))]
    pos += torch.randint(0, 3 * slots, (B - len(pos),), generator=g).tolist()
    check(pos[::-1] if B == 1 else pos, 8, 128, 2, window, sinks, slots, cuda, torch.bfloat16, TOL)


@pytest.mark.gpu
def test_gpu_strided_and_repeated(cuda):
    """A ring that is a slice of a larger one, and the same call twice."""
    big = torch.zeros(3, 60, 2 * 2 * 64 + 64, device=cuda, dtype=torch.bfloat16)
    qkv, ring, t, o = check([5, 49, 300], 4, 64, 2, 40, 4, 50, cuda, torch.bfloat16, TOL,
                            cache=big[:, 3:53, 32:32 + 256])
    again = ops.window_attention_step(qkv, ring, t, 4, 64, 2, window=40, sinks=4)
    assert torch.equal(o, again)
    wide = torch.cat([qkv, qkv], 1)[:, :qkv.shape[1]]
    assert torch.equal(o, ops.window_attention_step(wide, ring, t, 4, 64, 2, window=40, sinks=4))


@pytest.mark.gpu
def test_gpu_positions_and_offsets_past_32_bits(cuda):
    """A position past 2^32, and a ring whose last sequence starts past 2^31 elements."""
    H, hd, Hkv, window, sinks, slots = 4, 64, 2, 30, 2, 32
    p = (1 << 33) + 5
    qkv, ring, hist = case([64], H, hd, Hkv, window, sinks, slots, cuda, torch.bfloat16)
    # the same ring as at position 64, turned to where p finds it
    held = torch.arange(64 - window + 1, 64, device=cuda)
    far = torch.full_like(ring, math.nan)
    far[:, :sinks] = ring[:, :sinks]
    far[0, ops.ring_slot(held - 64 + p, sinks, slots)] = hist[0][held]
    near = ops.window_attention_step(qkv, ring, torch.tensor([64], device=cuda), H, hd, Hkv,
                                     window=window, sinks=sinks)
    got = ops.window_attention_step(qkv, far, torch.tensor([p], device=cuda), H, hd, Hkv,
                                    window=window, sinks=sinks)
    # the same rows in another order: sums differ by fp32 rounding, then bf16
    assert bool(((near.double() - got.double()).abs() <= 2.0**-8 * near.abs().double() + 2.0**-12).all())
    width = 2 * Hkv * hd
    rows = (1 << 31) // width + 64
    cache = torch.empty(3, rows, width, device=cuda, dtype=torch.bfloat16)
    qkv = torch.randn(3, H * hd + width, device=cuda).to(torch.bfloat16)
    last = rows - 10
    cache[2, last - 29:last] = torch.randn(29, width, device=cuda).to(torch.bfloat16)
    cache[2, :2] = torch.randn(2, width, device=cuda).to(torch.bfloat16)
    o = ops.window_attention_step(qkv, cache, torch.tensor([-1, -1, last], device=cuda), H, hd, Hkv,
                                  window=window, sinks=sinks)
    kv = torch.cat([cache[2, :2], cache[2, last - 29:last + 1]]).double().view(-1, 2, Hkv, hd)
    q = qkv[2, :H * hd].double().view(Hkv, -1, hd)
    w = torch.softmax(q @ kv[:, 0].permute(1, 2, 0) / math.sqrt(hd), -1)
    want = (w @ kv[:, 1].transpose(0, 1)).reshape(-1)
    assert torch.equal(cache[2, last], qkv[2, H * hd:])
    assert bool(((o[2].double() - want).abs() <= TOL * (want.abs() + 1.0)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("S,sinks,slots", [(1, 0, 4), (40, 4, 20), (40, 4, 64), (300, 0, 128)])
def test_gpu_fill(cuda, S, sinks, slots):
    B, H, hd, Hkv = 4, 4, 64, 2
    qkv = torch.randn(B * S, (H + 2 * Hkv) * hd, device=cuda).to(torch.bfloat16)
    n = torch.tensor([S, 0, max(1, S // 2), S + 9], dtype=torch.int32)
    for lengths in (None, n):
        ring = torch.zeros(B, slots, 2 * Hkv * hd, device=cuda, dtype=torch.bfloat16)
        host = ring.cpu().float()
        ops.window_cache_fill(qkv, ring, B, S, H, hd, Hkv, sinks=sinks,
                              lengths=None if lengths is None else lengths.to(cuda))
        ops.window_cache_fill(qkv.cpu().float(), host, B, S, H, hd, Hkv, sinks=sinks, lengths=lengths)
        assert torch.equal(ring.cpu().float(), host)


@pytest.mark.gpu
def test_gpu_refusals(cuda):
    def args(H=4, hd=64, Hkv=2, B=2, slots=8):
        return [torch.zeros(B, (H + 2 * Hkv) * hd, device=cuda, dtype=torch.bfloat16),
                torch.zeros(B, slots, 2 * Hkv * hd, device=cuda, dtype=torch.bfloat16),
                torch.zeros(B, device=cuda, dtype=torch.int64), H, hd, Hkv]

    step = ops.window_attention_step
    a = args()
    for kw in (dict(window=0), dict(window=4, sinks=-1), dict(window=4, sinks=8)):
        with pytest.raises(RuntimeError):
            step(*a, **kw)
    with pytest.raises(RuntimeError, match="head width"):
        step(*args(hd=48), window=4)
    with pytest.raises(RuntimeError, match="int64"):
        step(a[0], a[1], a[2].int(), *a[3:], window=4)
    with pytest.raises(RuntimeError, match="bf16"):
        step(a[0].float(), *a[1:], window=4)
    with pytest.raises(RuntimeError, match="cache must be"):
        step(a[0], a[1][:, :, :-8], *a[2:], window=4)
    with pytest.raises(RuntimeError, match="must be on"):
        step(a[0], a[1].cpu(), *a[2:], window=4)
    odd = torch.zeros(2 * a[0].shape[1] + 1, device=cuda, dtype=torch.bfloat16)[1:].view(2, -1)
    with pytest.raises(RuntimeError, match="aligned"):
        step(odd, *a[1:], window=4)
    none = args(B=0)
    assert step(*none, window=4).shape == (0, 256)

"""Counter-based dropout with the residual sum.

Would fail if: the words differed from the published generator or between the
host and the GPU; the mask depended on strides, alignment, type or direction;
a dropped element passed anything on; or a bad argument were taken.
"""

import pytest
import torch

from elysium_wan_b200 import ops


def philox_np(block, seed, stream):
    """Philox4x32-10 by its definition, one block, in Python integers."""
    c = [block & 0xFFFFFFFF, block >> 32, stream & 0xFFFFFFFF, stream >> 32]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def test_words_published_vectors():
    # the known answers that the generator's authors publish
    assert philox_np(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    assert philox_np(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    for seed, stream in ((0, 0), (12345, 7), (ones, ones - 3), (1 << 40, 1 << 33)):
        want = sum((philox_np(b, seed, stream) for b in range(5)), [])[:18]
        assert ops.dropout_words(18, seed, stream).tolist() == want


def test_host_path_mask_and_scale():
    x, r = torch.randn(37, 19), torch.randn(37, 19)
    y = ops.dropout_add(x, r, 0.25, 3, 9)
    keep = ops.dropout_words(x.numel(), 3, 9).view(x.shape) >= round(0.25 * 2**32)
    assert torch.equal(y, torch.where(keep, x * (1 / 0.75), 0.0) + r)
    assert torch.equal(ops.dropout_bwd(x, 0.25, 3, 9), torch.where(keep, x * (1 / 0.75), 0.0))
    # 703 draws of rate 0.75: six standard deviations are 0.098
    assert abs(keep.float().mean().item() - 0.75) < 0.098
    assert not torch.equal(ops.dropout_words(64, 3, 9), ops.dropout_words(64, 3, 10))
    assert torch.equal(ops.dropout_add(x, None, 0.0, 3, 9), x)


def test_host_path_gradient_is_the_difference_quotient():
    # the map is linear in x, so a difference quotient is exact up to fp64 rounding
    x, g = torch.randn(5, 7), torch.randn(5, 7)
    h = torch.randn(5, 7)
    d = (ops.dropout_add(x + h, None, 0.5, 1, 2) - ops.dropout_add(x, None, 0.5, 1, 2)).double()
    assert abs((d * g).sum() - (ops.dropout_bwd(g, 0.5, 1, 2).double() * h).sum()) < 1e-4


@pytest.mark.parametrize("p,seed,stream", [(1.0, 0, 0), (-0.1, 0, 0), (float("nan"), 0, 0),
                                           (0.1, -1, 0), (0.1, 0, 1 << 64)])
def test_refusals(p, seed, stream):
    with pytest.raises(ValueError):
        ops.dropout_add(torch.zeros(2, 2), None, p, seed, stream)


def test_refuses_shapes():
    with pytest.raises(ValueError):
        ops.dropout_add(torch.zeros(2, 2), torch.zeros(2, 3), 0.1, 0, 0)


def plain64(x, resid, p, seed, stream):
    keep = ops.dropout_words(x.numel(), seed, stream, x.device).view(x.shape)
    keep = keep >= min(round(p * 2**32), 2**32 - 1)
    y = torch.where(keep, x.double() / (1 - p), 0.0)
    return y if resid is None else y + resid.double()


# One rounding of the sum and one of the scale (fp32), then one to the output:
# half a unit in the last place of the output plus 2 fp32 roundings of the
# terms, taken together with room for the sum's cancellation.
def check(y, want, *terms):
    unit = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}[y.dtype]
    size = sum(t.double().abs() for t in terms)
    assert bool(((y.double() - want).abs() <= want.abs() * unit * 1.01 + 2.0**-22 * size + 1e-7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 7), (3, 8), (5, 13), (64, 768), (33, 1000), (2, 40001)])
@pytest.mark.parametrize("xt,rt,yt", [(torch.bfloat16, torch.bfloat16, torch.bfloat16),
                                      (torch.bfloat16, torch.float16, torch.float32),
                                      (torch.float32, torch.float32, torch.float32),
                                      (torch.float32, torch.bfloat16, torch.float16),
                                      (torch.bfloat16, None, torch.bfloat16)])
def test_gpu_against_plain(cuda, rows, d, xt, rt, yt):
    torch.manual_seed(rows * d)
    x = torch.randn(rows, d, device=cuda).to(xt)
    r = torch.randn(rows, d, device=cuda).to(rt) if rt else None
    seed, stream = (1 << 45) + 17, (1 << 35) + rows
    y = ops.dropout_add(x, r, 0.3, seed, stream, out_dtype=yt)
    assert y.dtype == yt
    terms = [x / 0.7] + ([r] if r is not None else [])
    check(y, plain64(x, r, 0.3, seed, stream), *terms)
    # the host path drops the same elements
    host = ops.dropout_add(x.cpu().float(), None, 0.3, seed, stream)
    assert torch.equal((ops.dropout_bwd(x, 0.3, seed, stream).cpu() != 0), (host != 0))


@pytest.mark.gpu
def test_gpu_strides_and_alignment(cuda):
    """Row strides and bases of every alignment draw the same mask."""
    for rows, d in ((5, 24), (4, 13), (7, 64)):
        big = torch.randn(rows, d + 40, device=cuda).to(torch.bfloat16)
        rbig = torch.randn(rows, d + 16, device=cuda).to(torch.bfloat16)
        for a in (0, 8, 3):
            x, r = big[:, a:a + d], rbig[:, a % 8:a % 8 + d]
            y = ops.dropout_add(x, r, 0.5, 5, 6)
            assert y.is_contiguous()
            assert torch.equal(y, ops.dropout_add(x.contiguous(), r.contiguous(), 0.5, 5, 6))
            check(y, plain64(x, r, 0.5, 5, 6), x * 2, r)


@pytest.mark.gpu
def test_gpu_dropped_nan_and_empty(cuda):
    x = torch.full((4, 64), float("nan"), device=cuda, dtype=torch.bfloat16)
    r = torch.ones(4, 64, device=cuda, dtype=torch.bfloat16)
    y = ops.dropout_add(x, r, 0.5, 1, 1)
    keep = ops.dropout_words(256, 1, 1).view(4, 64) >= 1 << 31
    assert torch.equal(torch.isnan(y).cpu(), keep)
    assert bool((y.cpu()[~keep] == 1).all())
    assert ops.dropout_add(x[:0], None, 0.5, 1, 1).shape == (0, 64)
    assert ops.dropout_add(x[:, :0], None, 0.5, 1, 1).shape == (4, 0)


@pytest.mark.gpu
def test_gpu_past_32_bits(cuda):
    """Elements past 2^32: the block counter's upper word and 64-bit offsets."""
    rows, d = 65537, 65536  # 2^32 + 65536 elements
    x = torch.ones(1, d, device=cuda, dtype=torch.bfloat16).expand(rows, d)
    y = ops.dropout_bwd(x, 0.5, 11, 12)
    for e in (0, (1 << 32) - 4, 1 << 32, (1 << 32) + 65532):
        want = [2.0 if w >= 1 << 31 else 0.0 for w in philox_np(e // 4, 11, 12)]
        assert y.view(-1)[e:e + 4].tolist() == want


@pytest.mark.gpu
def test_gpu_refusals(cuda):
    x = torch.zeros(4, 8, device=cuda, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="resid must have"):
        ops.dropout_add(x, x[:2], 0.1, 0, 0)
    with pytest.raises(RuntimeError, match="bf16 or fp32"):
        ops.dropout_add(x.half(), None, 0.1, 0, 0)
    with pytest.raises(RuntimeError, match="2-D"):
        ops.dropout_add(x[0], None, 0.1, 0, 0)
    with pytest.raises(RuntimeError, match="contiguous inner"):
        ops.dropout_add(x.t(), None, 0.1, 0, 0)
    with pytest.raises(RuntimeError, match="must be on"):
        ops.dropout_add(x, x.cpu(), 0.1, 0, 0)
    with pytest.raises(ValueError):
        ops.dropout_add(x, None, 1.0, 0, 0)


@pytest.mark.gpu
def test_gpu_other_stream(cuda):
    s = torch.cuda.Stream()
    x = torch.randn(512, 768, device=cuda).to(torch.bfloat16)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.dropout_add(x, x, 0.1, 4, 5)
    s.synchronize()
    assert torch.equal(y, ops.dropout_add(x, x, 0.1, 4, 5))

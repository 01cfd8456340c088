"""Calls of ``nvk_rotary`` that ``ops.rotary`` does not make, against the formula in 64 bits (see test_rotary_gpu), and
its angles against exact ones."""

import math

import pytest
import torch

from nano_vllm_ascend_b200 import _lib, ops
from tests.test_rotary_gpu import HALF, check, formula, frequencies

pytestmark = pytest.mark.gpu


# whole vectors of eight and of two elements, and element by element
@pytest.mark.parametrize("dim,rotated", [(128, 64), (20, 12), (130, 66)])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("weights", ["neither", "query's", "key's", "both"])
@pytest.mark.parametrize("has", ["query", "key"])
def test_weights_of_an_absent_side_are_not_used(cuda_device, has, weights, interleaved, dim, rotated):
    """With heads of q or of k alone, that side's weight says whether it is normed, and the other side's pointers are
    not looked at."""
    dev, t, h = cuda_device, 7, 3
    g = torch.Generator().manual_seed(dim)
    x = torch.randn(t, h, dim, generator=g).to(torch.bfloat16).to(dev)
    w = (1 + 0.3 * torch.randn(2, dim, generator=g)).to(torch.bfloat16).to(dev)
    inv, pos = frequencies(rotated // 2).to(dev), torch.randint(0, 1000, (t,), generator=g).to(dev)
    out, side = torch.full_like(x, float("nan")), int(has == "key")
    given = [weights in ("query's", "both"), weights in ("key's", "both")]

    def two(mine):  # (q's, k's) arguments
        return (0, mine) if side else (mine, 0)

    _lib.call("nvk_rotary", *two(out.data_ptr()), *two(x.data_ptr()), *two(h * dim), *two(h * dim),
              *(w[i].data_ptr() if given[i] else 0 for i in (0, 1)), 1e-6, inv.data_ptr(), pos.data_ptr(), 1.0, t,
              *two(h), dim, rotated, interleaved, 0, torch.cuda.current_stream(dev).cuda_stream)
    want, mag = formula(x, w[side] if given[side] else None, 1e-6, inv, pos, bool(interleaved), 1.0)
    check(out, want, mag)


PI = 31415926535897932384626433832795028841971693993751058209749445923078164062862089986280348253421170679  # times 10^-100


def exact_angles(positions, inv):
    """cos and sin of position * frequency [T, half], and the angles, from whole numbers."""
    bits = 256
    per_turn = (10 ** 100 << bits) // (2 * PI)  # 2^bits / (2 pi)
    cos, sin, angle = [], [], []
    for p in positions.tolist():
        for f in inv.tolist():
            m, d = f.as_integer_ratio()  # d a power of two
            part = (p * m * per_turn) % (d << bits)  # of a turn, times d 2^bits
            x = part / (d << bits) * 2 * math.pi
            cos.append(math.cos(x))
            sin.append(math.sin(x))
            angle.append(abs(p) * f)
    return (torch.tensor(t, dtype=torch.float64).view(len(positions), -1) for t in (cos, sin, angle))


@pytest.mark.parametrize("top", [1, 12, 24, 28, 30, 36, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_an_angle_is_off_by_what_the_header_says(cuda_device, top, dtype):
    """Turned rows (1, 0) against exact angles: the results near 0 (a few 2^-13 among so many) round by next to nothing,
    so that the angle's own error shows. 2^-26 of a turn, 2^-52 of the angle, and in fp32 the cosine (2^-23)
    and the product (2^-24)."""
    half, t = 64, 2000
    g = torch.Generator().manual_seed(top)
    positions = torch.randint(-(1 << top), 1 << top, (t,), generator=g)
    positions[0] = (1 << top) - 1
    inv = frequencies(half)
    x = torch.zeros(t, 1, 2 * half, dtype=dtype, device=cuda_device)
    x[..., :half] = 1
    got, _ = ops.rotary(x, x, inv.to(cuda_device), positions.to(cuda_device))
    cos, sin, angle = exact_angles(positions, inv)
    want = torch.cat((cos, sin), -1)
    off = 2 * math.pi * 2.0 ** -26 + angle * 2.0 ** -52 + 2.0 ** -23 + 2.0 ** -24
    err = (got[:, 0].double().cpu() - want).abs()
    tol = want.abs() * HALF[dtype] + torch.cat((off, off), -1) + 2.0 ** -25 * (dtype == torch.float16)
    assert bool((err <= tol).all()), float((err / tol).max())
    assert top < 12 or float(want.abs().min()) < 2.0 ** -13

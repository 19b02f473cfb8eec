"""The 8-bit cache's codes and scales, without a tolerance: codes are quotients of whole numbers rounded to the nearest,
halves to the even one, and scales the largest magnitude over 127, rounded once."""

import pytest
import torch

import chord_b200

pytestmark = pytest.mark.gpu


def written(rows, device):
    cache = chord_b200.kv_cache(len(rows), 1, 1, rows.shape[1], dtype=torch.uint8, device=device)
    rows = rows.to(device)
    chord_b200.cache_write(rows[:, None], -rows[:, None], cache, torch.arange(len(rows), dtype=torch.int32, device=device))
    chord_b200.check_status(device)
    return cache


def test_every_quotient(device):
    """All pairs of BF16 significands, x down to 2^-9 of the largest: (127 a) / (b 2^m) with a, b in 128..255."""
    a = torch.arange(128, 256)
    x = (a[None, :] * 2.0 ** -torch.arange(10)[:, None]).flatten()            # [10 * 128]
    numerator, shift = a.repeat(10) * 127, torch.arange(10).repeat_interleave(128)
    parts = [slice(i, i + 128) for i in range(0, 1280, 128)]
    rows, want = [], []
    for b in range(128, 256):
        denominator = b << shift
        whole, rest = numerator // denominator, numerator % denominator
        up = (2 * rest > denominator) | ((2 * rest == denominator) & (whole % 2 == 1))
        code = whole + up
        for p in parts:
            keep = x[p] <= b
            rows.append(torch.cat([torch.where(keep, x[p], 0.0), torch.full((128,), float(b))]))
            want.append(torch.where(keep, code[p], 0))
    rows, want = torch.stack(rows), torch.stack(want)
    exact = rows.to(torch.bfloat16)
    assert torch.equal(exact.float(), rows)
    for power in (-118, -110, 0, 60, 115):
        cache = written((rows.double() * 2.0 ** power).to(torch.bfloat16), device)
        for codes, sign in ((cache.k, 1), (cache.v, -1)):
            got = sign * (codes[:, 0, 0].int().cpu() - 128)
            assert torch.equal(got[:, :128].long(), want) and bool((got[:, 128:] == 127).all()), power


@pytest.mark.parametrize("dim", [16, 128, 256])
def test_scales_are_rounded_once(device, dim):
    tops = torch.arange(1, 0x7F80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    rows = torch.zeros((len(tops), dim), dtype=torch.bfloat16)
    rows[:, dim // 3] = tops
    cache = written(rows, device)
    want = tops.float() / 127
    assert torch.equal(cache.k_scale[:, 0, 0].cpu(), want) and torch.equal(cache.v_scale[:, 0, 0].cpu(), want)
    assert bool((cache.k[:, 0, 0, dim // 3] == 255).all()) and bool((cache.v[:, 0, 0, dim // 3] == 1).all())

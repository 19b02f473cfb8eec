"""`qk_norm_rope`, and the paged cache as it is written and read back, against 64 bits."""

import pytest
import torch

import chord_b200
from tests import attention_cases as A

pytestmark = pytest.mark.gpu


def heads_case(device, tokens, heads, kv_heads, dim, rotary, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    qkv = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=g, device=device).to(torch.bfloat16)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    qw, kw = (torch.rand(dim, generator=g, device=device).add(0.5).to(torch.bfloat16) for _ in range(2))
    table = A.angles(300, rotary, device)
    positions = torch.randint(0, 300, (tokens,), generator=g, device=device, dtype=torch.int32)
    return q, k, v, qw, kw, table, positions


def check(got, want, x, weight, table, positions, eps, interleaved):
    """One rounding to BF16, and some thirty roundings of FP32 on terms no larger than the head's largest."""
    limit = A.HALF * want.abs() + 32 * A.SINGLE * want.abs().amax(-1, keepdim=True) * 2 + 1e-38
    assert bool(((got.double() - want).abs() <= limit).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary", [
    (1, 64, 8, 128, 128), (3, 1, 1, 16, 16), (7, 5, 5, 64, 32), (2, 6, 2, 80, 48), (5, 12, 3, 96, 96), (4, 7, 1, 112, 0),
    (9, 16, 2, 192, 64), (3, 8, 4, 256, 256), (1000, 28, 4, 128, 64), (700, 9, 3, 64, 64), (600, 8, 8, 256, 128),
])
def test_norm_rope(device, tokens, heads, kv_heads, dim, rotary, interleaved):
    q, k, _, qw, kw, table, positions = heads_case(device, tokens, heads, kv_heads, dim, rotary, tokens)
    got = chord_b200.qk_norm_rope(q, k, qw, kw, table, positions, eps=1e-5, interleaved=interleaved)
    for x, w, out in ((q, qw, got[0]), (k, kw, got[1])):
        want = A.norm_rope(x, w, table, positions, 1e-5, interleaved)
        assert out.shape == x.shape and out.is_contiguous()
        check(out, want, x, w, table, positions, 1e-5, interleaved)


def test_norms_of_nothing_and_of_infinities(device):
    q, k, _, qw, kw, table, positions = heads_case(device, 3, 2, 2, 64, 64)
    q, k = q.clone(), k.clone()
    q[0] = 0
    q[1, 0, 5] = float("nan")
    q[1, 1, 6] = float("inf")
    a, b = chord_b200.qk_norm_rope(q, k, qw, kw, table, positions)
    assert bool((a[0] == 0).all())
    assert bool(torch.isnan(a[1, 0]).all())
    assert bool(torch.isnan(a[1, 1]).any())   # inf / inf
    check(a[2:], A.norm_rope(q[2:], qw, table, positions[2:], 1e-6, False), None, None, None, None, None, None)
    check(b, A.norm_rope(k, kw, table, positions, 1e-6, False), None, None, None, None, None, None)


def test_in_place(device):
    q, k, _, qw, kw, table, positions = heads_case(device, 700, 8, 2, 128, 128)
    want = chord_b200.qk_norm_rope(q, k, qw, kw, table, positions)
    q, k = q.contiguous(), k.contiguous()
    got = chord_b200.qk_norm_rope(q, k, qw, kw, table, positions, q_out=q, k_out=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_positions_outside_the_table(device):
    q, k, _, qw, kw, table, positions = heads_case(device, 4, 3, 1, 128, 64)
    positions[1], positions[2] = 300, -1
    chord_b200.check_status(device)
    a, b = chord_b200.qk_norm_rope(q, k, qw, kw, table, positions)
    assert bool((a[1:3] == 0).all()) and bool((b[1:3] == 0).all()) and bool((a[0] != 0).any())
    with pytest.raises(RuntimeError, match="outside"):
        chord_b200.check_status(device)
    chord_b200.check_status(device)


def cache_like(device, pages, page, heads, dim, bits, layout="heads"):
    if layout == "heads":
        return chord_b200.kv_cache(pages, page, heads, dim, dtype=torch.uint8 if bits == 8 else torch.bfloat16, device=device)
    dtype = torch.uint8 if bits == 8 else torch.bfloat16
    k, v = (torch.zeros((pages, page, heads, dim), dtype=dtype, device=device).transpose(1, 2) for _ in range(2))
    scales = [torch.zeros((pages, page, heads), device=device).transpose(1, 2) for _ in range(2)] if bits == 8 else []
    return chord_b200.KVCache(k, v, *scales)


def check_kept(got, x, bits, exact_input=True):
    """What comes back: the BF16 value itself, or half a step (and FP32's roundings) away and rounded to
    BF16."""
    x = x.double()
    if bits == 16:
        if exact_input:
            assert torch.equal(got.double(), x)
            return
        step = torch.zeros_like(x[..., :1])
    else:
        step = x.abs().amax(-1, keepdim=True) / 127
    limit = 0.5 * step * (1 + 2.0 ** -12) + A.HALF * x.abs() + A.HALF * 0.5 * step + 64 * A.SINGLE * x.abs().amax(-1, keepdim=True)
    assert bool(((got.double() - x).abs() <= limit).all())


@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("lengths,page,heads,dim", [
    ([1], 1, 1, 16), ([5, 0, 9], 4, 3, 64), ([17, 31, 1], 16, 2, 96), ([40], 24, 5, 128), ([3, 50, 7, 0], 7, 4, 192),
    ([129, 64], 64, 8, 256), ([900, 1, 1200], 32, 8, 128), ([2], 100, 2, 112),
])
def test_write_and_read_back(device, lengths, page, heads, dim, bits, layout):
    g = torch.Generator().manual_seed(sum(lengths))
    total = sum(lengths)
    pages = sum(-(-n // page) for n in lengths) + 2
    cache = cache_like(device, pages, page, heads, dim, bits, layout)
    table = A.tables_for(lengths, page, pages, g, extra=1)
    k, v = (torch.randn((total, heads, dim), generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    slots = torch.tensor([int(table[b, t // page]) * page + t % page for b, n in enumerate(lengths) for t in range(n)],
                         dtype=torch.int32)
    offsets = torch.tensor([0] + list(torch.tensor(lengths).cumsum(0)), dtype=torch.int32)
    chord_b200.cache_write(k, v, cache, slots.to(device))
    rows = total + 3
    k_out, v_out = (torch.full((rows, heads, dim), float("nan"), dtype=torch.bfloat16, device=device) for _ in range(2))
    chord_b200.cache_read(cache, table.to(device), offsets.to(device), rows, k_out=k_out, v_out=v_out)
    chord_b200.check_status(device)
    for got, x in ((k_out, k), (v_out, v)):
        check_kept(got[:total], x, bits)
        assert bool((got[total:] == 0).all())
    # pages that no slot named are as they were
    kept = torch.zeros(pages * page, dtype=torch.bool)
    kept[slots.long()] = True
    assert bool((cache.k.transpose(1, 2).reshape(pages * page, heads, dim)[~kept.to(device)] == 0).all())


@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary", [(1, 8, 2, 128, 128), (61, 28, 4, 128, 64), (13, 5, 5, 64, 16),
                                                              (4, 12, 1, 192, 192), (800, 16, 4, 256, 256)])
def test_norm_rope_write(device, tokens, heads, kv_heads, dim, rotary, interleaved, bits):
    q, k, v, qw, kw, table, positions = heads_case(device, tokens, heads, kv_heads, dim, rotary, tokens + bits)
    page = 16
    pages = -(-tokens // page) + 1
    cache = cache_like(device, pages, page, kv_heads, dim, bits)
    g = torch.Generator().manual_seed(1)
    blocks = A.tables_for([tokens], page, pages, g)
    slots = (blocks[0, torch.arange(tokens) // page] * page + torch.arange(tokens) % page).to(torch.int32).to(device)
    got_q = chord_b200.qk_norm_rope_write(q, k, v, qw, kw, table, positions, cache, slots, interleaved=interleaved)
    same_q, _ = chord_b200.qk_norm_rope(q, k, qw, kw, table, positions, interleaved=interleaved)
    assert torch.equal(got_q, same_q)
    got = chord_b200.cache_read(cache, blocks.to(device), torch.tensor([0, tokens], dtype=torch.int32, device=device), tokens)
    check_kept(got[0], A.norm_rope(k, kw, table, positions, 1e-6, interleaved), bits, exact_input=False)
    check_kept(got[1], v, bits)


def test_slots_and_pages_outside(device):
    cache = cache_like(device, 3, 4, 2, 64, 8)
    k, v = (torch.randn((4, 2, 64), device=device).to(torch.bfloat16) for _ in range(2))
    chord_b200.check_status(device)
    chord_b200.cache_write(k, v, cache, torch.tensor([-1, 5, -7, 2], dtype=torch.int32, device=device))
    chord_b200.check_status(device)      # negative: not kept, no mistake
    assert int((cache.k_scale != 0).sum()) == 4
    chord_b200.cache_write(k, v, cache, torch.tensor([12, 2**31 - 1, 0, 1], dtype=torch.int32, device=device))
    with pytest.raises(RuntimeError, match="outside"):
        chord_b200.check_status(device)
    assert int((cache.k_scale != 0).sum()) == 8
    offsets = torch.tensor([0, 9], dtype=torch.int32, device=device)
    a, _ = chord_b200.cache_read(cache, torch.tensor([[0, 3]], dtype=torch.int32, device=device), offsets, 9)
    with pytest.raises(RuntimeError, match="outside"):
        chord_b200.check_status(device)      # page 3, and a third page that the table lacks
    assert bool((a[:3] != 0).any()) and bool((a[4:] == 0).all())


def test_rows_of_zeros_infinities_and_tiny_values(device):
    cache = cache_like(device, 1, 8, 1, 64, 8)
    x = torch.randn((6, 1, 64), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(device)
    x[1] = 0
    x[2, 0, 3] = float("inf")
    x[3, 0, 9] = float("nan")
    x[4] *= 2.0 ** -118
    x[5] *= 2.0 ** 120
    chord_b200.cache_write(x, x, cache, torch.arange(6, dtype=torch.int32, device=device))
    zero = torch.zeros((1, 1), dtype=torch.int32, device=device)
    got, _ = chord_b200.cache_read(cache, zero, torch.tensor([0, 6], dtype=torch.int32, device=device), 6)
    assert bool((got[1] == 0).all()) and bool(torch.isnan(got[2:4]).all())
    for i in (0, 4, 5):
        check_kept(got[i:i + 1], x[i:i + 1], 8)


def test_halves_go_to_the_even_code(device):
    """A row's largest x is 127 steps, so +-x / 2 is 63.5 steps: 64; for every size of x, the type's largest too.
    The other columns are n + 1/2 steps where the largest is 127 or 254 of something: all n.  No tolerance."""
    tops = torch.arange(1 << 7, 0x7F80, dtype=torch.int32, device=device).to(torch.int16).view(torch.bfloat16)
    tops = tops[tops >= 2.0 ** -120]
    n = torch.arange(127, device=device).float()
    rows = torch.stack([tops, tops / 2, -tops / 2] + [torch.zeros_like(tops)] * 253, dim=1)
    steps = torch.zeros((40, 256), device=device)
    steps[:, :127], steps[:, 127], steps[:, 128:255] = n + 0.5, 127, -n - 0.5
    steps *= 2.0 ** torch.arange(-100, 100, 5, device=device).float()[:, None]
    x = torch.cat([rows, steps.to(torch.bfloat16)])
    cache = chord_b200.kv_cache(len(x), 1, 1, 256, dtype=torch.uint8, device=device)
    chord_b200.cache_write(x[:, None], -x[:, None], cache, torch.arange(len(x), dtype=torch.int32, device=device))
    even = torch.round(n + 0.5)   # (torch rounds halves to even)
    for codes, sign in ((cache.k[:, 0, 0], 1), (cache.v[:, 0, 0], -1)):
        codes = sign * (codes.int() - 128)
        head, tail = codes[:len(rows)], codes[len(rows):]
        assert bool((head[:, 0] == 127).all()) and bool((head[:, 1] == 64).all()) and bool((head[:, 2] == -64).all())
        assert bool((head[:, 3:] == 0).all())
        assert bool((tail[:, :127] == even).all()) and bool((tail[:, 128:255] == -even).all())
    for scale, x in ((cache.k_scale, x), (cache.v_scale, -x)):
        want = x.double().abs().amax(1) / 127
        assert bool(((scale[:, 0, 0].double() - want).abs() <= 4 * A.SINGLE * want).all())
    chord_b200.check_status(device)


@pytest.mark.parametrize("bits", [8, 16])
def test_a_cache_past_four_gigabytes(device, bits):
    """Offsets of the last pages pass 2^32 bytes."""
    heads, dim, page = 8, 256, 64
    pages = (5 << 30) // (heads * dim * page * (2 if bits == 16 else 1))
    cache = cache_like(device, pages, page, heads, dim, bits)
    x, y = (torch.randn((2, heads, dim), generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).to(device) for s in (1, 2))
    slots = torch.tensor([pages * page - 1, 3], dtype=torch.int32, device=device)
    chord_b200.cache_write(x, y, cache, slots)
    table = torch.tensor([[pages - 1], [0]], dtype=torch.int32, device=device)
    got = chord_b200.cache_read(cache, table, torch.tensor([0, page, page + 4], dtype=torch.int32, device=device), page + 4)
    for out, want in zip(got, (x, y)):
        check_kept(out[[page - 1, page + 3]], want, bits)
    chord_b200.check_status(device)


def test_refusals(device):
    q, k, v, qw, kw, table, positions = heads_case(device, 3, 4, 2, 64, 64)
    call = chord_b200.qk_norm_rope
    with pytest.raises(TypeError, match="q must be"):
        call(q.float(), k, qw, kw, table, positions)
    with pytest.raises(ValueError, match="k must have shape"):
        call(q, k[:2], qw, kw, table, positions)
    with pytest.raises(TypeError, match="q_weight"):
        call(q, k, qw.float(), kw, table, positions)
    with pytest.raises(ValueError, match="columns"):
        call(q, k, qw, kw, table[:, :40].contiguous(), positions)
    with pytest.raises(TypeError, match="positions"):
        call(q, k, qw, kw, table, positions.long())
    with pytest.raises(ValueError, match="positions"):
        call(q, k, qw, kw, table, positions[:2])
    with pytest.raises(ValueError, match="eps"):
        call(q, k, qw, kw, table, positions, eps=-1.0)
    with pytest.raises(TypeError, match="interleaved"):
        call(q, k, qw, kw, table, positions, interleaved=1)
    with pytest.raises(ValueError, match="q_out"):
        call(q, k, qw, kw, table, positions, q_out=q)      # a view with gaps
    with pytest.raises(ValueError, match="16-byte"):
        call(q[..., 1:17], k[..., 1:17], qw[:16], kw[:16], table[:, :16].contiguous(), positions)
    cache = cache_like(device, 2, 8, 2, 64, 16)
    slots = torch.zeros(3, dtype=torch.int32, device=device)
    with pytest.raises(TypeError, match="KVCache"):
        chord_b200.cache_write(k, v, cache.k, slots)
    with pytest.raises(ValueError, match="shape"):
        chord_b200.cache_write(q, v, cache, slots)
    with pytest.raises(ValueError, match="slots"):
        chord_b200.cache_write(k, v, cache, slots[:2])
    with pytest.raises(ValueError, match="block_tables"):
        chord_b200.cache_read(cache, slots.view(1, 3), slots, 3)
    with pytest.raises(ValueError, match="total"):
        chord_b200.cache_read(cache, slots.view(1, 3), slots[:2], -1)
    with pytest.raises(ValueError, match="k_out"):
        chord_b200.cache_read(cache, slots.view(1, 3), slots[:2], 2, k_out=k)
    assert chord_b200.qk_norm_rope(q[:0], k[:0], qw, kw, table, positions[:0])[0].shape == (0, 4, 64)
    chord_b200.cache_write(k[:0], v[:0], cache, slots[:0])

"""`gemv` against the product in 64 bits from checkpoint codes."""

import pytest
import torch

import chord_b200
from tests import attention_cases as A
from tests.cases import make_weights

pytestmark = pytest.mark.gpu


def check(got, want, size, k):
    """One rounding to BF16, and K / 16 + K / 32 + 32 additions of FP32."""
    limit = A.HALF * want.abs() + (k / 16 + k / 32 + 32) * A.SINGLE * size
    assert bool(((got.double() - want).abs() <= limit * 1.001 + 1e-38).all()), float(((got.double() - want).abs() - limit).max())


def weight_of(experts, n, k, seed, device, **scales):
    codes, scale = make_weights(experts, n, k, seed, **scales)
    codes, scale = codes.to(device), scale.to(device)
    return codes, scale, chord_b200.pack_w4a16(codes, scale)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 13, 16])
@pytest.mark.parametrize("n,k", [(128, 64), (256, 512), (384, 192), (128, 4160), (1024, 2048)])
def test_dense(device, rows, n, k):
    codes, scale, weight = weight_of(1, n, k, 7 * rows + n, device)
    x = torch.randn((rows, k), generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16).to(device)
    got = chord_b200.gemv(x, weight)
    want, size = A.gemv(x, codes, scale)
    assert got.shape == (rows, n)
    check(got, want, size, k)
    again = chord_b200.gemv(x, weight)
    assert torch.equal(got, again)


@pytest.mark.parametrize("n,k", [(4096, 7168), (7168, 2048), (128, 14336), (14336, 256)])
@pytest.mark.parametrize("rows", [1, 6, 16])
def test_large(device, rows, n, k):
    codes, scale, weight = weight_of(1, n, k, rows, device)
    x = torch.randn((rows, k), generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).to(device)
    want, size = A.gemv(x, codes, scale)
    check(chord_b200.gemv(x, weight), want, size, k)


@pytest.mark.parametrize("rows", [1, 2, 4, 7])
def test_more_blocks_than_are_resident(device, rows):
    """300 blocks of 64 weight rows: CTAs of four warps, with batches of K left over."""
    n, k = 19200, 1344
    codes, scale, weight = weight_of(1, n, k, rows, device)
    x = torch.randn((rows, k), generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).to(device)
    want, size = A.gemv(x, codes, scale)
    check(chord_b200.gemv(x, weight), want, size, k)


def test_experts_of_more_blocks_than_are_resident(device):
    experts, n, k, rows = 5, 640, 576, 40
    codes, scale, weight = weight_of(experts, n, k, 3, device)
    g = torch.Generator().manual_seed(4)
    x = torch.randn((rows, k), generator=g).to(torch.bfloat16).to(device)
    ids = torch.randint(0, 7, (rows,), generator=g, dtype=torch.int32)
    got = chord_b200.gemv(x, weight, expert_ids=ids.to(device))
    for e in range(7):
        mine = (ids == e).nonzero()[:, 0].to(device)
        if e >= experts:
            assert bool((got[mine] == 0).all())
        elif len(mine):
            want, size = A.gemv(x[mine], codes[e:e + 1], scale[e:e + 1])
            check(got[mine], want, size, k)


@pytest.mark.parametrize("rows", [2, 6])
def test_results_at_an_odd_element(device, rows):
    """A result needs no more alignment than its type; rows of experts held elsewhere are zeros there too."""
    n, k = 256, 320
    codes, scale, weight = weight_of(2, n, k, 8, device)
    x = torch.randn((rows, k), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(device)
    ids = torch.tensor([1, 5] * (rows // 2), dtype=torch.int32, device=device)
    room = torch.full((rows * n + 2,), 7.0, dtype=torch.bfloat16, device=device)
    out = room[1:-1].view(rows, n)
    chord_b200.gemv(x, weight, expert_ids=ids, outputs=out)
    want, size = A.gemv(x[::2], codes[1:], scale[1:])
    check(out[::2], want, size, k)
    assert bool((out[1::2] == 0).all()) and float(room[0]) == float(room[-1]) == 7.0


@pytest.mark.parametrize("tokens,top_k", [(1, 1), (1, 8), (3, 2), (5, 7)])
@pytest.mark.parametrize("base", [0, 3])
def test_experts(device, tokens, top_k, base):
    experts, n, k = 9, 256, 448
    codes, scale, weight = weight_of(experts, n, k, tokens, device)
    g = torch.Generator().manual_seed(tokens + base)
    x = torch.randn((tokens, k), generator=g).to(torch.bfloat16).to(device)
    ids = torch.randint(0, 16, (tokens, top_k), generator=g, dtype=torch.int32)  # some held elsewhere
    ids[0, 0] = base
    local = ids.flatten().long() - base
    local = torch.where((local >= 0) & (local < experts), local, -1)
    out = torch.full((tokens * top_k, n), float("nan"), dtype=torch.bfloat16, device=device)
    got = chord_b200.gemv(x, weight, expert_ids=ids.to(device), top_k=top_k, expert_base=base, outputs=out)
    assert got is out
    want, size = A.gemv(x, codes, scale, local, top_k)
    check(got, want, size, k)
    assert bool((got[(local < 0).to(device)] == 0).all())


def test_experts_far_apart(device):
    """Offsets of the last expert pass 2^31 words' bytes."""
    n, k, experts = 1024, 2048, 2100  # 1024 * 2048 / 2 bytes each: 2.2 GB
    words = torch.randint(-2**31, 2**31 - 1, (experts, k // 16, 2 * n), dtype=torch.int32, device=device)
    scale = torch.full((experts, k // 32, n), 0.01, dtype=torch.bfloat16, device=device)
    weight = chord_b200.PreparedWeight(packed=words, scale=scale, n=n, k=k, num_experts=experts)
    x = torch.randn((1, k), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(device)
    ids = torch.tensor([experts - 1, 0], dtype=torch.int32, device=device)
    got = chord_b200.gemv(x, weight, expert_ids=ids, top_k=2)
    for row, e in enumerate((experts - 1, 0)):
        alone = chord_b200.PreparedWeight(packed=words[e:e + 1].clone(), scale=scale[e:e + 1], n=n, k=k, num_experts=1)
        assert torch.equal(got[row:row + 1], chord_b200.gemv(x, alone))


def test_strided_rows_and_streams(device):
    codes, scale, weight = weight_of(1, 256, 320, 3, device)
    wide = torch.randn((5, 2 * 320 + 6), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(device)
    x = wide[:, 322:642]
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        got = chord_b200.gemv(x, weight)
    torch.cuda.current_stream(device).wait_stream(stream)
    want, size = A.gemv(x, codes, scale)
    check(got, want, size, 320)


def test_infinities_and_scales(device):
    """An infinity in x meets weights of both signs and of zero, as in the plain product; scales of every
    size count in full."""
    n, k = 128, 256
    codes, scale, _ = weight_of(1, n, k, 11, device)
    scale = scale * 2.0 ** torch.randint(-60, 60, scale.shape, generator=torch.Generator().manual_seed(4)).to(device)
    scale = scale.to(torch.bfloat16)
    weight = chord_b200.pack_w4a16(codes, scale)
    x = torch.randn((2, k), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(device)
    want, size = A.gemv(x, codes, scale)
    check(chord_b200.gemv(x, weight), want, size, k)
    x[1, 37] = float("inf")
    got = chord_b200.gemv(x, weight)
    check(got[:1], want[:1], size[:1], k)
    sign = (codes[0, :, 37] - 8).sign().double()
    expected = torch.where(sign == 0, float("nan"), sign * float("inf"))
    assert torch.equal(torch.isnan(got[1]), torch.isnan(expected))
    assert torch.equal(got[1].double().nan_to_num(nan=0.0, posinf=1, neginf=-1), sign)
    x[1, 37] = float("nan")
    assert bool(torch.isnan(chord_b200.gemv(x, weight)[1]).all())


def test_agrees_with_indexed(device):
    """The same weight through `indexed`, whose weights are rounded to BF16: three roundings of 2^-8."""
    experts, n, k = 4, 256, 512
    codes, scale, weight = weight_of(experts, n, k, 21, device)
    x = torch.randn((3, k), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(device)
    ids = torch.tensor([[0, 2], [3, 1], [2, 3]], dtype=torch.int32, device=device)
    block_m = chord_b200.indexed_block_m(weight, 3, 2)
    routing = chord_b200.moe_align_block_size(ids, block_m, experts)
    a, b = chord_b200.gemv(x, weight, expert_ids=ids, top_k=2), chord_b200.indexed(x, weight, *routing, 2, block_m=block_m)
    _, size = A.gemv(x, codes, scale, ids.flatten().cpu(), 2)
    assert bool(((a.double() - b.double()).abs() <= 2 * A.HALF * a.double().abs() + A.HALF * size).all())


def test_replays_from_a_graph(device):
    codes, scale, weight = weight_of(1, 512, 1024, 13, device)
    x = torch.zeros((2, 1024), dtype=torch.bfloat16, device=device)
    chord_b200.gemv(x, weight)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chord_b200.gemv(x, weight)
    x.copy_(torch.randn((2, 1024), generator=torch.Generator().manual_seed(9)))
    graph.replay()
    assert torch.equal(out, chord_b200.gemv(x, weight))


def test_refusals(device):
    _, _, weight = weight_of(2, 128, 64, 1, device)
    _, _, one = weight_of(1, 128, 64, 1, device)
    x = torch.zeros((2, 64), dtype=torch.bfloat16, device=device)
    ids = torch.zeros(2, dtype=torch.int32, device=device)
    with pytest.raises(TypeError, match="x must be"):
        chord_b200.gemv(x.float(), one)
    with pytest.raises(TypeError, match="PreparedWeight"):
        chord_b200.gemv(x, one.packed)
    with pytest.raises(ValueError, match="K=32"):
        chord_b200.gemv(x[:, :32], one)
    with pytest.raises(ValueError, match="expert_ids"):
        chord_b200.gemv(x, weight)
    with pytest.raises(ValueError, match="at most 16"):
        chord_b200.gemv(x.repeat(9, 1), one)
    with pytest.raises(ValueError, match="top_k"):
        chord_b200.gemv(x, one, top_k=2)
    with pytest.raises(ValueError, match="4 values"):
        chord_b200.gemv(x, weight, expert_ids=ids, top_k=2)
    with pytest.raises(TypeError, match="expert_ids"):
        chord_b200.gemv(x, weight, expert_ids=ids.long())
    with pytest.raises(ValueError, match="contiguous rows"):
        chord_b200.gemv(torch.zeros((64, 2), dtype=torch.bfloat16, device=device).t(), one)
    with pytest.raises(ValueError, match="outputs"):
        chord_b200.gemv(x, one, outputs=torch.zeros((2, 64), dtype=torch.bfloat16, device=device))
    assert chord_b200.gemv(x[:0], one).shape == (0, 128)

"""The short ways through the wrappers of the operators over the paged cache give what the wrappers give, and leave to
them what is not plain."""

import pytest
import torch

import chord_b200
from chord_b200 import _lib
from tests import attention_cases as A

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, device, bits):
        g = torch.Generator(device=device).manual_seed(1)
        self.cache = chord_b200.kv_cache(40, 16, 2, 64, dtype=bits, device=device)
        A.fill(self.cache, g)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
        self.table = torch.arange(32, dtype=torch.int32, device=device).view(2, 16)
        self.new_table = torch.arange(32, 40, dtype=torch.int32, device=device).view(2, 4)
        self.lengths, self.offsets, self.groups = ints([200, 77]), ints([0, 3, 7]), ints([0, 1, 2])
        self.q = torch.randn((7, 8, 64), generator=g, device=device).to(torch.bfloat16)
        self.slopes = torch.rand(8, generator=g, device=device)
        self.starts, self.prefixes = ints([0, 0, 5, 0, 3, 3, 3]), ints([10, 20])
        self.lse = torch.zeros((2, 8), device=device)
        self.weights = torch.rand((2, 2, 256), generator=g, device=device)


@pytest.fixture
def both(device, monkeypatch):
    if _lib.direct() is None:
        pytest.skip("the module was not built")
    chord_b200.indexed_gemm.status_word(device)
    chord_b200.indexed_gemm.default_locks(device)
    module = _lib.direct()

    def run(name, call):
        taken = []
        spy = type("Spy", (), {n: staticmethod(getattr(module, n)) for n in dir(module) if not n.startswith("_")})
        setattr(spy, name, staticmethod(lambda *args: taken.append(getattr(module, name)(*args)) or taken[-1]))
        with monkeypatch.context() as m:
            m.setattr(_lib, "direct", lambda: spy)
            a = call()
        assert len(taken) == 1 and taken[0] is not None  # (the short way was taken)
        with monkeypatch.context() as m:
            m.setattr(_lib, "direct", lambda: None)
            b = call()
        for x, y in zip(*((r if isinstance(r, tuple) else (r,)) for r in (a, b))):
            assert x.shape == y.shape and x.stride() == y.stride() and x.dtype == y.dtype and torch.equal(x, y)
        return a

    return run


@pytest.mark.parametrize("bits", [torch.bfloat16, torch.uint8])
def test_results_agree(device, both, bits):
    c = Case(device, bits)
    for options in (dict(cap=5.0), dict(slopes=c.slopes, window=9), dict(cap=30.0, scale=0.3, lse=c.lse)):
        both("paged_attention_shaped", lambda: chord_b200.paged_attention(c.q[:2], c.cache, c.table, c.lengths, **options))
        both("shared_prefix_attention", lambda: chord_b200.shared_prefix_attention(c.q[:2], c.cache, c.table, c.lengths, c.groups, c.new_table,
                                                                                   c.lengths // 4, **options))
    for options in ({}, dict(cap=5.0), dict(slopes=c.slopes, window=9, starts=c.starts), dict(prefixes=c.prefixes, lse=torch.empty((7, 8), device=device))):
        both("prompt_attention", lambda: chord_b200.prompt_attention(c.q, c.cache, c.table, c.lengths, c.offsets, **options))
    for options in ({}, dict(cap=5.0), dict(slopes=c.slopes, window=9)):
        both("attention_weights", lambda: chord_b200.attention_weights(c.q[:2], c.cache, c.table, c.lengths, c.lse, **options))
    both("attention_weights", lambda: chord_b200.attention_weights(c.q[:2], c.cache, c.table, c.lengths, c.lse, weights=c.weights.clone()))
    given = c.weights.clone()
    assert chord_b200.attention_weights(c.q[:2], c.cache, c.table, c.lengths, c.lse, weights=given) is given
    both("cache_evict", lambda: chord_b200.cache_evict(c.cache, c.table, c.lengths, c.weights, 50, first=2, recent=3, new_tables=c.new_table))
    both("cache_evict", lambda: chord_b200.cache_evict(c.cache, c.table, c.lengths, c.weights, 300))
    chord_b200.check_status(device)


def test_what_is_left_to_the_wrapper(device, both):
    module, c = _lib.direct(), Case(device, torch.bfloat16)
    at = (c.cache.address, c.cache.index)
    long = 1 << 80
    calls = {
        module.prompt_attention: ([c.q, *at, c.table, c.lengths, c.offsets, None, None, None, 0.1, None, None, None],
                                  ((0, c.q[:, :3]), (0, c.q[:0]), (0, c.q.float()), (3, c.table[:1]), (3, c.table.long()), (4, c.lengths[:1]),
                                   (5, c.offsets[:1]), (5, c.offsets.long()), (5, c.offsets[::2]), (6, c.starts[:3]), (7, c.starts), (8, c.lse),
                                   (9, 1), (9, float("inf")), (10, 0), (10, -1), (10, 2.0), (10, long), (10, True), (11, 0.0), (11, -1.0), (11, 5),
                                   (11, float("nan")), (12, c.slopes[:3]), (12, c.slopes.double()), (2, 63))),
        module.shared_prefix_attention: ([c.q[:2], *at, c.table, c.lengths, c.groups, c.new_table, c.lengths // 4, None, 0.1, None, None, None],
                                         ((0, c.q), (3, c.table[:1]), (4, c.lengths[:1]), (5, c.groups[:1]), (6, c.table[:1]), (7, c.starts),
                                          (8, c.slopes), (9, 1), (10, 0), (11, 0.0), (12, c.lse))),
        module.paged_attention_shaped: ([c.q[:2], *at, c.table, c.lengths, None, 0.1, None, 5.0, None],
                                        ((0, c.q), (3, c.table[:1]), (4, c.starts), (5, c.slopes), (6, 1), (7, 0), (8, 0.0), (9, c.lse))),
        module.attention_weights: ([c.q[:2], *at, c.table, c.lengths, c.lse, None, 0.1, None, None, None],
                                   ((0, c.q), (3, c.table[:1]), (4, c.starts), (5, None), (5, c.slopes), (6, c.weights[:1]), (6, c.weights[..., ::2]),
                                    (6, c.weights.double()), (7, 1), (8, 0), (9, 0.0), (10, c.lse))),
        module.cache_evict: ([*at, c.table, c.lengths, c.weights, 50, 2, 3, None],
                             ((2, c.table[:1]), (3, c.lengths.long()), (3, c.lengths[:0]), (4, c.weights[:1]), (4, c.weights[..., ::2]), (5, 0), (5, 4),
                              (5, long), (5, 50.0), (6, -1), (6, 48), (7, -1), (7, True), (8, c.table[:1]), (8, c.new_table[:, :2]))),
    }
    for call, (args, wrongs) in calls.items():
        assert call(*args) is not None
        assert call(*args[:-1]) is None
        for place, value in wrongs:
            wrong = list(args)
            wrong[place] = value
            assert call(*wrong) is None, (call, place, value)
    chord_b200.check_status(device)

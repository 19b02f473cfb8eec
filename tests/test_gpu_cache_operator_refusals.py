"""What the wrappers of the operators over prompts, shared prefixes and evictions refuse, before anything is launched; and
what only looks as if it should be."""

import math

import pytest
import torch

import chord_b200

pytestmark = pytest.mark.gpu


class Calls:
    """Good arguments of each operator; a call with some of them changed."""

    def __init__(self, device):
        self.cache = chord_b200.kv_cache(8, 16, 2, 64, device=device)
        for x in (self.cache.k, self.cache.v):
            x.normal_()
        self.q = torch.randn((4, 6, 64), device=device).bfloat16()
        ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
        self.table, self.one = ints(*range(8)).reshape(4, 2), ints(7, 6).reshape(1, 2)
        self.lengths, self.lse = ints(5, 0, 17, 32), torch.zeros((4, 6), device=device)
        self.weights = torch.rand((4, 2, 40), device=device)
        self.good = {
            "prompt_attention": dict(q=self.q, cache=self.cache, block_tables=self.table[:2].contiguous(), lengths=ints(20, 9), offsets=ints(0, 3, 4)),
            "shared_prefix_attention": dict(q=self.q, cache=self.cache, prefix_tables=self.one, prefix_lengths=ints(30),
                                            group_offsets=ints(0, 4), block_tables=self.table, lengths=self.lengths),
            "attention_weights": dict(q=self.q, cache=self.cache, block_tables=self.table, lengths=self.lengths, lse=self.lse),
            "cache_evict": dict(cache=self.cache, block_tables=self.table, lengths=self.lengths, weights=self.weights, keep=8),
            "paged_attention": dict(q=self.q, cache=self.cache, block_tables=self.table, lengths=self.lengths),
        }

    def __call__(self, name, **changes):
        return getattr(chord_b200, name)(**{**self.good[name], **changes})


SCORED = ["prompt_attention", "shared_prefix_attention", "attention_weights", "paged_attention"]


@pytest.mark.parametrize("name", SCORED)
def test_scores(device, name):
    call = Calls(device)
    for change, message in (({"scale": math.nan}, "scale"), ({"scale": True}, "scale"), ({"scale": "1"}, "scale"), ({"window": 0}, "window"),
                            ({"window": 2**31}, "window"), ({"window": 1.5}, "window"), ({"cap": 0.0}, "cap"), ({"cap": -3.0}, "cap"),
                            ({"cap": math.inf}, "cap"), ({"cap": 1e-31}, "cap"), ({"cap": 1e-3, "scale": 1e36}, "cap"),
                            ({"slopes": torch.zeros(5, device=device)}, "slopes"), ({"slopes": torch.zeros(6)}, "slopes"),
                            ({"slopes": torch.zeros(12, device=device)[::2]}, "slopes")):
        with pytest.raises((ValueError, RuntimeError), match=message):
            call(name, **change)
    with pytest.raises(TypeError, match="slopes"):
        call(name, slopes=torch.zeros(6, device=device, dtype=torch.float64))
    call(name)
    call(name, cap=1e30, scale=1, window=2**31 - 1)
    chord_b200.check_status(device)


@pytest.mark.parametrize("name", SCORED)
def test_queries_and_tables(device, name):
    call = Calls(device)
    for q in (call.q.float(), call.q[0], None):
        with pytest.raises(TypeError, match="q must"):
            call(name, q=q)
    for q in (call.q.cpu(), call.q[..., :48], call.q.transpose(1, 2), call.q[:, :5], torch.zeros((4, 6, 65), dtype=torch.bfloat16, device=device)[..., 1:]):
        with pytest.raises(ValueError):
            call(name, q=q)
    with pytest.raises(TypeError, match="block_tables"):
        call(name, block_tables=call.table.long())
    for table in (call.table[:1], call.table.cpu(), call.table[0]):
        with pytest.raises((ValueError, TypeError), match="block_tables"):
            call(name, block_tables=table)
    with pytest.raises(TypeError, match="lengths"):
        call(name, lengths=call.lengths.long())
    with pytest.raises(ValueError, match="lengths"):
        call(name, lengths=call.lengths[:1])
    rows = call.good[name]["q"].shape[0]
    for lse in (torch.zeros((rows, 5), device=device), torch.zeros((rows, 6)), torch.zeros((6, rows), device=device).t()):
        with pytest.raises(ValueError, match="lse"):
            call(name, lse=lse)
    with pytest.raises(TypeError, match="lse"):
        call(name, lse=torch.zeros((rows, 6), device=device, dtype=torch.float64))
    call(name)
    chord_b200.check_status(device)


def test_what_is_written_lies_apart(device):
    call = Calls(device)
    memory = torch.zeros(8192, dtype=torch.float32, device=device)
    q = memory[:768].view(torch.bfloat16).reshape(4, 6, 64)
    for name in ("prompt_attention", "shared_prefix_attention"):
        with pytest.raises(ValueError, match="lse must not overlap q"):
            call(name, q=q, lse=memory[700:724].reshape(4, 6))
        with pytest.raises(ValueError, match="outputs must not overlap q"):
            call(name, q=q, outputs=q)
        with pytest.raises(ValueError, match="lse must not overlap outputs"):
            call(name, outputs=q, lse=memory[700:724].reshape(4, 6))
        call(name, q=q, lse=memory[768:792].reshape(4, 6))
    lse = memory[4000:4024].reshape(4, 6)
    with pytest.raises(ValueError, match="weights must not overlap lse"):
        call("attention_weights", lse=lse, weights=memory[3990:4310].reshape(4, 2, 40))
    with pytest.raises(ValueError, match="weights must not overlap q"):
        call("attention_weights", q=q, weights=memory[700:1020].reshape(4, 2, 40))
    chord_b200.check_status(device)


def test_weights(device):
    call = Calls(device)
    memory = torch.zeros(8192, dtype=torch.float32, device=device)
    for name in ("attention_weights", "cache_evict"):
        with pytest.raises(TypeError, match="weights"):
            call(name, weights=call.weights.double())
        for wrong in (call.weights[:3], call.weights[:, :1], call.weights[..., :0], call.weights.cpu(), call.weights[0],
                      memory.as_strided((4, 2, 40), (200, 100, 2))):
            with pytest.raises(ValueError, match="weights"):
                call(name, weights=wrong)
    for strides in ((0, 40, 1), (40, 40, 1), (80, 0, 1), (40, 20, 1), (60, 40, 1), (40, 140, 1)):
        with pytest.raises(ValueError, match="overlap"):
            call("attention_weights", weights=memory.as_strided((4, 2, 40), strides))
    for strides in ((80, 40, 1), (40, 160, 1), (100, 50, 1)):  # either order of sequences and heads, with room between
        to = memory.zero_().as_strided((4, 2, 40), strides)
        assert call("attention_weights", lse=call.lse, weights=to) is to
        assert torch.equal(to[..., :32], call("attention_weights", lse=call.lse))
        assert int(memory.count_nonzero()) == int(to.count_nonzero())
    with pytest.raises(TypeError, match="lse"):
        call("attention_weights", lse=None)
    chord_b200.check_status(device)


def test_evictions(device):
    call = Calls(device)
    for change, message in (({"keep": 0}, "keep"), ({"keep": 2.0}, "keep"), ({"keep": True}, "keep"), ({"keep": 2**28}, "keep"), ({"first": -1}, "first"),
                            ({"recent": -1}, "recent"), ({"first": 5, "recent": 4}, "first"),
                            ({"new_tables": call.table[:, :1].contiguous(), "keep": 17}, "new_tables")):
        with pytest.raises(ValueError, match=message):
            call("cache_evict", **change)
    with pytest.raises(TypeError, match="new_tables"):
        call("cache_evict", new_tables=call.table.long())
    for lengths in (call.lengths.reshape(2, 2), call.lengths.long(), None):
        with pytest.raises(TypeError, match="lengths"):
            call("cache_evict", lengths=lengths)
    chord_b200.check_status(device)


def test_groups_and_offsets(device):
    call = Calls(device)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    for name, argument in (("prompt_attention", "offsets"), ("shared_prefix_attention", "group_offsets")):
        with pytest.raises(TypeError, match=argument):
            call(name, **{argument: i(0, 4).long()})
        for wrong in (i(0), i(0, 4).reshape(1, 2), i(0, 4).cpu()):
            with pytest.raises(ValueError, match=argument):
                call(name, **{argument: wrong})
    with pytest.raises(ValueError, match="starts"):
        call("prompt_attention", starts=i(0, 0, 0))
    with pytest.raises(ValueError, match="prefixes"):
        call("prompt_attention", prefixes=i(0))
    with pytest.raises(ValueError, match="prefix_lengths"):
        call("shared_prefix_attention", prefix_lengths=i(1, 2))
    with pytest.raises(ValueError, match="prefix_tables"):
        call("shared_prefix_attention", prefix_tables=call.table)
    chord_b200.check_status(device)

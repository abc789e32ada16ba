"""CPU: what the Python calls of the serving steps refuse before the library
sees it. Without a context the library itself answers BH_EINVAL, so a call that
gets past the wrappers' own checks shows as a BHError."""
from __future__ import annotations

import types

import pytest
import torch


class On(torch.Tensor):
    """A tensor that says it lies on a GPU."""

    index = 0

    is_cuda = property(lambda t: True)

    def get_device(self):
        return self.index

    @property
    def device(self):
        return torch.device("cuda", self.index)


def on(index, t):
    t = torch.Tensor._make_subclass(On, t)
    t.index = index
    return t


@pytest.fixture(autouse=True)
def default_stream(bh, monkeypatch):
    """Without a GPU there is no current stream to ask for."""
    monkeypatch.setattr(bh, "_raw_stream", lambda device: 0)


CTX = types.SimpleNamespace(h=None, device=0)
WS = types.SimpleNamespace(h=None)


def step(bh, away):
    """One call of each operator, the tensor called `away` on another GPU than the rest."""
    def at(name, t):
        return on(1 if name == away else 0, t)

    def ints(name, *shape, dtype=torch.int32):
        return at(name, torch.zeros(shape, dtype=dtype))

    cache_at = 1 if away == "cache" else 0
    cache = bh.PagedKV(on(cache_at, torch.zeros(4, 16, 2, 64)), on(cache_at, torch.zeros(4, 16, 2, 64)))
    plan_out = bh.KVPlan(ints("q_start", 2), ints("seq", 3), ints("pos", 3), ints("slot", 3, dtype=torch.int64),
                         ints("mask", 3, dtype=torch.int64), ints("counts", 2))
    q = at("q", torch.zeros(3, 4, 64))
    yield lambda: bh.kv_plan(CTX, ints("ctx_lens", 1), ints("new_lens", 1), ints("free_blocks", 4), ints("tables", 1, 4), 16, 3,
                             parents=ints("parents", 3), out=plan_out, stream=0)
    yield lambda: bh.qk_norm_rope_append(CTX, at("qkv", torch.zeros(3, 8 * 64)), 4, cache, at("rope", torch.zeros(8, 32, 2)),
                                         plan_out.pos, plan_out.slot, q_norm=at("q_norm", torch.zeros(64)),
                                         k_norm=at("k_norm", torch.zeros(64)), q_out=q, stream=0)
    yield lambda: bh.tree_attention(CTX, WS, q, cache, ints("tables", 1, 4), ints("ctx_lens", 1), plan_out.q_start, 3,
                                    mask=plan_out.mask, out=at("out", torch.zeros(3, 4, 64)), stream=0)
    if away in ("logits", "tokens", None):
        yield lambda: bh.token_logprobs(CTX, WS, at("logits", torch.zeros(2, 9)), ints("tokens", 2), 1, stream=0)


def test_calls_on_one_gpu_reach_the_library(bh):
    for call in step(bh, None):
        with pytest.raises(bh.BHError):
            call()


@pytest.mark.parametrize("away", ["ctx_lens", "new_lens", "free_blocks", "tables", "parents", "q_start", "seq", "pos", "slot", "mask",
                                  "counts", "qkv", "rope", "q_norm", "k_norm", "q", "out", "cache", "logits", "tokens"])
def test_a_tensor_of_another_gpu_is_refused(bh, away):
    refused = 0
    for call in step(bh, away):
        try:
            call()
        except ValueError:
            refused += 1
        except bh.BHError:
            pass
    assert refused == {"ctx_lens": 2, "tables": 2, "q_start": 2, "pos": 2, "slot": 2, "mask": 2, "q": 2, "cache": 2}.get(away, 1)


def test_a_cache_of_two_gpus_is_refused(bh):
    with pytest.raises(ValueError):
        bh.PagedKV(on(0, torch.zeros(4, 16, 2, 64)), on(1, torch.zeros(4, 16, 2, 64)))


@pytest.mark.parametrize("shape", [(8, 64, 4), (8, 64), (16, 32, 2, 2)])
def test_a_rotation_table_of_another_shape_is_refused(bh, shape):
    """Also one with enough values, which would be read as other angles."""
    cache = bh.PagedKV(on(0, torch.zeros(4, 16, 2, 64)), on(0, torch.zeros(4, 16, 2, 64)))
    with pytest.raises(ValueError):
        bh.qk_norm_rope_append(CTX, on(0, torch.zeros(3, 8 * 64)), 4, cache, on(0, torch.zeros(shape)), on(0, torch.zeros(3, dtype=torch.int32)),
                               on(0, torch.zeros(3, dtype=torch.int64)), stream=0)

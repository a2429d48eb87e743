"""Checks of the attention operators' Python calls that need no GPU: what is refused before a kernel could see it."""
from types import SimpleNamespace

import pytest
import torch

from loki_b200 import attention as A


class _NoCall:
    """Stands for the library: a refused call must not reach it."""

    def __getattr__(self, name):
        def fail(*_):
            raise AssertionError("%s was called" % name)
        return fail


@pytest.fixture()
def here():
    """A context, cache, rope table and arguments that share a device: -1, which is what host tensors report."""
    ctx = A.AttnContext.__new__(A.AttnContext)
    ctx.device, ctx._lib, ctx.ctx = -1, _NoCall(), None
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    return SimpleNamespace(ctx=ctx, cache=SimpleNamespace(device=-1, n_seqs=1, dtype=torch.bfloat16, _ref=None),
                           table=SimpleNamespace(device=-1, rot_dim=64, max_pos=16, address=0), i32=i32, bf=bf,
                           calls=lambda c, cache, table, **k: {
                               "rope": lambda: c.rope(bf(2, 3, 64), i32(2), table, **k),
                               "append": lambda: c.append(cache, bf(2, 512), bf(2, 64), i32(2), i32(2), table, **k),
                               "tree": lambda: c.tree(bf(2, 3, 576), cache, i32(2), None, 0.1, **k),
                               "mass": lambda: c.mass(bf(2, 3, 576), torch.zeros(2, 3), cache, i32(2), None, 0.1, **k),
                               "evict": lambda: c.evict(cache, 4, i32(1), **k)})


@pytest.mark.parametrize("name", ["append", "tree", "mass", "evict"])
def test_a_cache_on_another_device_is_refused(here, name):
    here.cache.device = 1
    with pytest.raises(ValueError, match="cache"):
        here.calls(here.ctx, here.cache, here.table)[name]()


@pytest.mark.parametrize("name", ["rope", "append"])
def test_a_table_on_another_device_is_refused(here, name):
    here.table.device = 1
    with pytest.raises(ValueError, match="table"):
        here.calls(here.ctx, here.cache, here.table)[name]()


@pytest.mark.parametrize("name", ["rope", "append", "tree", "mass", "evict"])
def test_a_stream_of_another_device_is_refused(here, name):
    other = SimpleNamespace(device=torch.device("cuda", 1), cuda_stream=0)
    with pytest.raises(ValueError, match="stream"):
        here.calls(here.ctx, here.cache, here.table, stream=other)[name]()
    with pytest.raises(ValueError, match="stream"):
        here.ctx.device_error(other)

"""Caches in four bits: calls one after another that no other test makes."""
import pytest
import torch

from cake_b200.capi import CakeB200Error, check, lib
from cake_b200.model import Context, TextModelBase
from tests.test_packed_cache import EINVAL, ESTATE, rows
from tests.util import checkpoint, medium_config


@pytest.mark.gpu
def test_a_refused_begin_leaves_the_graph_refused():
    """Rows were written behind the decode graph's back; a begin that is refused does not make it runnable."""
    cfg = medium_config(num_hidden_layers=1)
    ctx = Context(cfg, checkpoint(cfg, "bf16", std=0.05, peaked=True), "bf16", cache_bits=4)
    m = TextModelBase.load(ctx)
    m.forward([[1, 2, 3, 4, 5, 6, 7, 8]], 0)
    m.index_pos = 8
    m.decode_build()
    m.decode_greedy(5, 2)
    k = rows(1, 3, 2, 64, "bf16", 1)
    ctx.cache.write(0, k, k, 6)
    for token, pos, code in ((cfg.vocab_size, 9, EINVAL), (5, 8, ESTATE)):
        with pytest.raises(CakeB200Error) as e:
            check(lib().cake_b200_decode_begin(ctx.h, token, pos))
        assert e.value.code == code
        with pytest.raises(CakeB200Error) as e:
            check(lib().cake_b200_decode_run(ctx.h, 1))
        assert e.value.code == ESTATE
    m.index_pos = 9
    assert len(m.decode_greedy(5, 2)) == 2 and ctx.cache.len(0) == 11
    ctx.close()

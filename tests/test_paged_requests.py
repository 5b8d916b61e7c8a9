"""Requests that run together over a cache in pages: more of them than one call of the head takes, some that fill their sequences, calls that fail."""
import numpy as np
import pytest
import torch

from oracle import oracle as O
from tests.test_gpu_parity import LOGIT_TOL_ULP, _ctx
from tests.util import checkpoint, max_ulp_err, medium_config, to_np


def model_for(cfg, dtype="bf16", max_seq=None, **kw):
    from cake_b200.model import TextModelBase
    return TextModelBase.load(_ctx(cfg, checkpoint(cfg, dtype, seed=17, **kw), dtype, max_seq=max_seq))


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [65, 150])
def test_more_requests_than_the_head_takes_at_once(requests):
    """Each request has the logits and the token of its own prompt, wherever it stands in the step."""
    from cake_b200.model import PagedSessions
    cfg = medium_config()
    sd = checkpoint(cfg, "bf16", seed=17)
    om, m = O.OracleModel(cfg, sd, "bf16"), model_for(cfg)
    g = np.random.default_rng(5)
    kinds = [[int(t) for t in g.integers(0, cfg.vocab_size, n)] for n in (1, 2, 3, 5, 9, 1, 4)]
    caches = [om.new_cache() for _ in kinds]
    ses = PagedSessions(m, 2 * requests, 16, max_requests=requests)
    at = [0] * len(kinds)
    feed = kinds
    for _ in range(3):
        want = [om.forward(np.array(x, np.uint32), p, c) for x, p, c in zip(feed, at, caches)]
        at = [p + len(x) for p, x in zip(at, feed)]
        best = {}
        got = ses.step({str(i): feed[i % len(kinds)] for i in range(requests)}, best)
        m.ctx.sync()
        assert list(got) == [str(i) for i in range(requests)] == list(best)
        for i in range(requests):
            x = to_np(got[str(i)])
            assert max_ulp_err(x, want[i % len(kinds)], "bf16") <= LOGIT_TOL_ULP
            assert best[str(i)] == int(x.argmax())
        feed = [[int(w.argmax())] for w in want]
    m.ctx.close()

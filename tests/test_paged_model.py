"""Models whose requests run together over a cache in pages, against the oracle and against the same requests one by one over caches of their own."""
import random

import numpy as np
import pytest
import torch

from cake_b200.capi import CakeB200Error
from cake_b200.synth import residual_deltas
from oracle import oracle as O
from tests.test_gpu_parity import CONFIGS, LOGIT_TOL_ULP, SIBLINGS, _ctx
from tests.util import checkpoint, max_ulp_err, medium_config, to_np

pytestmark = pytest.mark.gpu


def model_for(cfg, dtype, **kw):
    from cake_b200.model import TextModelBase
    ctx = _ctx(cfg, checkpoint(cfg, dtype, seed=17, **kw), dtype)
    return TextModelBase.load(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("name", [n for n in CONFIGS if not n.startswith("ref_")])   # (heads of 64 entries)
def test_requests_together_match_the_oracle(name, dtype):
    """Prompts of several lengths, then tokens, late arrivals and leavers: each request's logits are those of the oracle for it alone."""
    from cake_b200.model import PagedSessions
    cfg = CONFIGS[name]()
    sd = checkpoint(cfg, dtype, seed=17)
    om, m = O.OracleModel(cfg, sd, dtype), model_for(cfg, dtype)
    ses = PagedSessions(m, 60, 16, max_requests=4)
    rng = random.Random(4)
    caches, at = {}, {}

    def ask(tokens):
        got = ses.step(tokens)
        m.ctx.sync()
        for rid, ids in tokens.items():
            if rid not in caches:
                caches[rid], at[rid] = om.new_cache(), 0
            want = om.forward(np.array(ids, np.uint32), at[rid], caches[rid])
            at[rid] += len(ids)
            assert ses.len(rid) == at[rid]
            e = max_ulp_err(to_np(got[rid]), want, dtype)
            assert e <= LOGIT_TOL_ULP, (rid, at[rid], e)

    def ids(n):
        return [rng.randrange(cfg.vocab_size) for _ in range(n)]

    ask({"a": ids(5), "b": ids(33), "c": ids(1)})
    for _ in range(3):
        ask({r: ids(1) for r in "abc"})
    ask({"b": ids(1), "d": ids(20), "a": ids(4)})
    ses.end("b")
    ask({"e": ids(3), "a": ids(1), "c": ids(1), "d": ids(2)})
    for r in "acde":
        ses.end(r)
    assert ses.cache.available == 60
    m.ctx.close()


def test_tokens_of_requests_together_are_those_of_each_alone():
    """Greedy generation, three requests in one batch and each over a cache of its own.  Either way's logits lie within LOGIT_TOL_ULP of the oracle's, so the two
    within twice that of one another, and their first places agree where the best two lie further apart than two such errors."""
    from cake_b200.model import Cache, PagedSessions
    from tests.util import ulp_at_scale
    cfg = medium_config(max_seq_len=256)
    m = model_for(cfg, "bf16", peaked=True)
    rng = random.Random(9)
    prompts = {r: [rng.randrange(cfg.vocab_size) for _ in range(n)] for r, n in (("x", 70), ("y", 3), ("z", 21))}
    alone, logits_alone, sure = {}, {}, 0
    for r, p in prompts.items():
        m.ctx.cache = Cache(m.ctx, 1)
        m.prepare_prompt(p)
        alone[r], logits_alone[r] = [], []
        for i in range(12):
            alone[r].append(m.next_token(i).id)
            logits_alone[r].append(to_np(m.last_logits))
    ses = PagedSessions(m, 30, 16, max_requests=3)
    feed = dict(prompts)
    for i in range(12):
        logits = ses.step(feed)
        m.ctx.sync()
        for r in prompts:
            got, want = to_np(logits[r]), logits_alone[r][i]
            assert max_ulp_err(got, want, "bf16") <= 2 * LOGIT_TOL_ULP
            top = np.sort(want)[-2:]
            if top[1] - top[0] > 4 * LOGIT_TOL_ULP * ulp_at_scale(want, "bf16"):
                sure += 1
                assert got.argmax() == alone[r][i]
            feed[r] = [alone[r][i]]
    assert sure >= 6
    m.ctx.close()


def test_steps_that_do_not_fit():
    """Pages run out, sequences grow too long, token ids are none: nothing has happened, and what fits goes on."""
    from cake_b200.model import PagedSessions
    cfg = medium_config()
    m = model_for(cfg, "bf16")
    ses = PagedSessions(m, 6, 16, max_requests=3, max_seq=64)
    first = ses.step({"a": list(range(30))})["a"].clone()
    for bad, code in (({"b": list(range(50)), "c": list(range(30))}, -5), ({"a": list(range(40))}, -4)):
        with pytest.raises(CakeB200Error) as e:
            ses.step(bad)
        assert e.value.code == code
        assert set(ses.live) == {"a"} and ses.len("a") == 30 and ses.cache.available == 4
    for bad in ({"a": [1], "b": [cfg.vocab_size]}, {"a": [-1]}):
        with pytest.raises((ValueError, OverflowError)):
            ses.step(bad)
        assert set(ses.live) == {"a"} and ses.len("a") == 30
    with pytest.raises(CakeB200Error):
        ses.step({"a": [1], "b": []})
    with pytest.raises(CakeB200Error):
        ses.step({})
    assert set(ses.live) == {"a"} and ses.len("a") == 30
    again = ses.step({"b": list(range(30))})["b"]
    m.ctx.sync()
    assert torch.equal(first, again)
    m.ctx.close()


@pytest.mark.parametrize("kind", list(SIBLINGS))
def test_sibling_blocks_in_pages(kind):
    """Norms behind the sublayers, windows and rotations of each layer's own: the blocks take the path of every batch."""
    from cake_b200.model import PagedSessions, TextModelBase
    cfg = medium_config(num_hidden_layers=4, **SIBLINGS[kind])
    sd = checkpoint(cfg, "bf16", seed=31)
    if cfg.residual_rms_norm:
        sd = residual_deltas(sd)
    om, ctx = O.OracleModel(cfg, sd, "bf16", max_seq=64), _ctx(cfg, sd, "bf16", max_seq=64)
    ses = PagedSessions(TextModelBase.load(ctx), 16, 16, max_requests=2)
    caches, at = {"a": om.new_cache(), "b": om.new_cache()}, {"a": 0, "b": 0}
    g = np.random.default_rng(3)
    for counts in ({"a": 9, "b": 2}, {"a": 1, "b": 1}, {"b": 3, "a": 1}, {"a": 1, "b": 4}, {"a": 2}, {"b": 1, "a": 1}):
        ids = {r: [int(x) for x in g.integers(0, cfg.vocab_size, n)] for r, n in counts.items()}
        got = ses.step(ids)
        ctx.sync()
        for r, x in ids.items():
            want = om.forward(np.array(x, np.uint32), at[r], caches[r])
            at[r] += len(x)
            assert max_ulp_err(to_np(got[r]), want, "bf16") <= LOGIT_TOL_ULP
    ctx.close()


def test_several_prompts_of_the_command_line(tmp_path):
    """``python -m cake_b200.run`` with prompts side by side: the tokens of ``PagedSessions.generate``, which are the first places of its steps' logits."""
    import subprocess
    import sys
    from cake_b200.model import PagedSessions
    from tests.test_cpp_host import _write_model
    cfg = medium_config(num_hidden_layers=2, max_seq_len=128)
    sd = checkpoint(cfg, "bf16", seed=17, peaked=True)
    _write_model(tmp_path, cfg, sd)
    m = model_for(cfg, "bf16", peaked=True)
    rng = random.Random(2)
    prompts = [[rng.randrange(cfg.vocab_size) for _ in range(n)] for n in (17, 1, 40)]
    ses = PagedSessions(m, 12, 16, max_requests=3)
    names = {str(i): p for i, p in enumerate(prompts)}
    got = ses.generate(names, 9)
    assert ses.cache.available == 12 and not ses.live
    feed = dict(names)
    for i in range(9):
        logits = ses.step(feed)
        m.ctx.sync()
        feed = {}
        for r in names:
            if i < len(got[r]):
                assert int(logits[r].float().argmax()) == got[r][i]
                feed[r] = [got[r][i]]
        if not feed:
            break
    assert max(map(len, got.values())) == 9
    m.ctx.close()
    run = subprocess.run([sys.executable, "-m", "cake_b200.run", str(tmp_path), "--prompt-ids", ";".join(",".join(map(str, p)) for p in prompts), "-n", "9"],
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    lines = run.stdout.splitlines()
    assert [[int(t) for t in line.split(":")[1].split()] for line in lines[:3]] == [got[r] for r in names]
    for bad in (["--prompt-ids", "1;;2"], ["--prompt-ids", "1;2", "--temperature", "0.5"], ["--prompt-ids", "1;2", "--cache-bits", "4"]):
        assert subprocess.run([sys.executable, "-m", "cake_b200.run", str(tmp_path), *bad], capture_output=True, timeout=300).returncode == 2


def test_a_wait_that_was_given_up_closes_the_cache_until_its_sequences_are_dropped():
    import ctypes
    from cake_b200.model import PagedSessions
    from tests.test_gpu_waits import probe
    cfg = medium_config(num_hidden_layers=1)
    m = model_for(cfg, "bf16")
    ses = PagedSessions(m, 20, 16, max_requests=2)
    first = ses.step({"a": [1, 2, 3]})["a"].clone()
    m.ctx.sync()
    ok, kcycles = (ctypes.c_int * 2)(), (ctypes.c_int * 2)()
    probe(m.ctx, 1, 8192, ok, kcycles)   # a probe kernel's wait for an arrival that nobody makes
    with pytest.raises(CakeB200Error, match="gave up a wait"):
        m.ctx.sync()
    for _ in range(2):
        with pytest.raises(CakeB200Error) as e:
            ses.step({"a": [4]})
        assert e.value.code == -4 and "gave up" in str(e.value)
        with pytest.raises(CakeB200Error):
            ses.step({"b": [4]})
    assert ses.len("a") == 3 and set(ses.live) == {"a"}
    ses.end("a")
    again = ses.step({"b": [1, 2, 3]})["b"]
    m.ctx.sync()
    assert torch.equal(first, again)
    m.ctx.close()

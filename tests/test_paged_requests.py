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


@pytest.mark.gpu
def test_a_step_that_the_blocks_refuse_is_none():
    """More new rows than the window on a sequence that has some, a cache of another context: sequences as before, and they go on."""
    from cake_b200.capi import CakeB200Error
    from cake_b200.model import PagedCache
    cfg = medium_config(sliding_window=5)
    m, other = model_for(cfg), model_for(cfg)
    pages = PagedCache(m.ctx, 12, 16, max_seqs=2)
    a, b = pages.add(), pages.add()
    m.forward_paged(pages, [(a, [3, 1, 4, 1])])
    free = pages.available
    with pytest.raises(CakeB200Error) as e:
        m.forward_paged(pages, [(b, [7] * 20), (a, [1, 5, 9, 2, 6, 5])])
    assert e.value.code == -1 and "window" in str(e.value)
    assert (pages.len(a), pages.len(b), pages.available) == (4, 0, free)
    with pytest.raises(CakeB200Error) as e:
        other.forward_paged(pages, [(a, [1]), (b, [2])])
    assert e.value.code == -1 and "context" in str(e.value)
    assert (pages.len(a), pages.len(b), pages.available) == (4, 0, free)
    got = m.forward_paged(pages, [(a, [1, 5]), (b, [2])])
    fresh = PagedCache(m.ctx, 12, 16, max_seqs=2)
    x, y = fresh.add(), fresh.add()
    m.forward_paged(fresh, [(x, [3, 1, 4, 1])])
    want = m.forward_paged(fresh, [(x, [1, 5]), (y, [2])])
    m.ctx.sync()
    assert torch.equal(got, want)
    other.ctx.close()
    m.ctx.close()


class Pages:
    """Lengths of sequences, for PagedSessions without a GPU."""

    def __init__(self, max_seq):
        self.max_seq, self.lens = max_seq, {}

    def add(self):
        s = next(i for i in range(99) if i not in self.lens)
        self.lens[s] = 0
        return s

    def drop(self, s):
        del self.lens[s]

    def len(self, s):
        return self.lens[s]


def sessions(max_seq, answer, eos=()):
    """PagedSessions in front of a model that answers a request of length n with answer(n); a sequence beyond max_seq fails the whole step, as the library does."""
    from types import SimpleNamespace
    from cake_b200.capi import CakeB200Error
    from cake_b200.model import PagedSessions
    ses = PagedSessions.__new__(PagedSessions)

    def forward(pages, requests, greedy):
        if any(pages.lens[s] + len(t) > pages.max_seq for s, t in requests):
            raise CakeB200Error(-4, "positions exceed max_seq")
        for s, t in requests:
            pages.lens[s] += len(t)
        greedy[:] = [answer(pages.lens[s]) for s, _ in requests]
        return [None] * len(requests)
    ses.model = SimpleNamespace(forward_paged=forward, ctx=SimpleNamespace(config=SimpleNamespace(is_eos=lambda t: t in eos)))
    ses.cache, ses.live = Pages(max_seq), {}
    return ses


def test_a_request_that_fills_its_sequence_ends_and_the_others_go_on():
    ses = sessions(64, lambda n: n)
    got = ses.generate({"long": [1] * 60, "short": [1] * 10, "full": [1] * 64}, 32)
    assert got == {"long": [60, 61, 62, 63, 64], "short": list(range(10, 42)), "full": [64]}
    assert not ses.live and not ses.cache.lens
    ses = sessions(64, lambda n: n, eos=(62,))
    assert ses.generate({"a": [1] * 60, "b": [1] * 63}, 9) == {"a": [60, 61], "b": [63, 64]}
    assert ses.generate({"a": [1] * 60}, 3) == {"a": [60, 61]} and ses.generate({"a": [1] * 60}, 1) == {"a": [60]} and ses.generate({"a": [1]}, 0) == {"a": []}
    assert not ses.live and not ses.cache.lens


def test_generation_begins_no_request_that_is_live():
    ses = sessions(64, lambda n: n)
    ses.step({"a": [1, 2, 3]}, {})
    with pytest.raises(ValueError):
        ses.generate({"b": [1], "a": [4]}, 5)
    assert list(ses.live) == ["a"] and ses.len("a") == 3
    assert ses.generate({"b": [1]}, 2) == {"b": [1, 2]}
    assert list(ses.live) == ["a"] and ses.len("a") == 3


@pytest.mark.gpu
def test_prompts_of_which_one_reaches_the_end_of_its_sequence():
    from cake_b200.model import PagedSessions
    cfg = medium_config()
    m = model_for(cfg, max_seq=64)
    g = np.random.default_rng(8)
    prompts = {r: [int(t) for t in g.integers(0, cfg.vocab_size, n)] for r, n in (("long", 60), ("short", 10))}
    got = PagedSessions(m, 8, 16, max_requests=2, max_seq=64).generate(prompts, 32)
    wide = PagedSessions(m, 8, 16, max_requests=2, max_seq=64)
    feed, best = dict(prompts), {}
    for i in range(5):
        wide.step(feed, best)
        assert [best[r] for r in prompts] == [got[r][i] for r in prompts]
        feed = {r: [best[r]] for r in prompts}
    wide.end("long")
    for i in range(5, 32):
        best = {}
        wide.step({"short": feed["short"]}, best)
        assert best["short"] == got["short"][i]
        feed = {"short": [best["short"]]}
    assert len(got["long"]) == 5 and len(got["short"]) == 32
    m.ctx.close()


@pytest.mark.gpu
def test_logits_are_read_on_the_callers_stream():
    """Behind work that the library's stream still has in front of the step, and again after their memory has been given back and taken by the next step."""
    from cake_b200.model import PagedSessions
    cfg = medium_config()
    m = model_for(cfg)
    ses = [PagedSessions(m, 12, 16, max_requests=2) for _ in range(2)]
    feeds = [{"a": [3, 1, 4], "b": [1, 5]}, {"a": [9]}, {"a": [2, 6], "b": [5]}]
    want = []
    for feed in feeds:
        got = ses[0].step(feed)
        m.ctx.sync()
        want.append({r: x.clone() for r, x in got.items()})
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            kept = []
            for feed in feeds:
                with torch.cuda.stream(m.ctx.torch_stream):
                    torch.cuda._sleep(30_000_000)   # some 15 ms
                got = ses[1].step(feed)
                torch.cuda._sleep(10_000_000)
                kept.append({r: x + 0 for r, x in got.items()})
                del got
        stream.synchronize()
        for w, k in zip(want, kept):
            assert all(torch.equal(w[r], k[r]) for r in w)
        for r in "ab":
            ses[1].end(r)
    m.ctx.close()


@pytest.mark.parametrize("prompts,n,eos,behind", [([3, 1], 5, (), 8), ([3, 1], 1, (), 0), ([3], 4, (5,), 2), ([3, 9], 6, (3, 9), 0), ([2], 0, (), 0), ([60, 1], 9, (), 12)])
def test_the_rate_of_requests_together_leaves_the_prompts_out(monkeypatch, prompts, n, eos, behind):
    """A clock on which a step takes 1 s and the prompts' step 100: tokens behind the first step's over the seconds since then."""
    from cake_b200 import model
    clock = [0.0]
    monkeypatch.setattr(model.time, "perf_counter", lambda: clock[0])
    ses = sessions(64, lambda n: n, eos)
    step = ses.step

    def timed(tokens, best):
        clock[0] += 100.0 if not any(ses.len(r) for r in tokens) else 1.0
        return step(tokens, best)
    monkeypatch.setattr(ses, "step", timed)
    ses.generate({str(i): [1] * x for i, x in enumerate(prompts)}, n)
    steps = clock[0] - 100.0 if n else 0.0
    assert ses.tok_s == (behind / steps if behind else 0.0)


def test_both_rates_of_the_command_line_are_of_one_kind(monkeypatch, tmp_path, capsys):
    """cake_b200.run prints what generate, or generate_text, counted, in the same line for one prompt and for several."""
    from types import SimpleNamespace
    from cake_b200 import build, loader, model, run
    cfg = medium_config()
    monkeypatch.setattr(loader, "open_model", lambda d: (cfg, {}))
    monkeypatch.setattr(build, "build", lambda **kw: None)
    monkeypatch.setattr(model, "Context", lambda *a, **kw: SimpleNamespace(close=lambda: None))
    monkeypatch.setattr(model.TextModelBase, "load", classmethod(lambda cls, ctx, **kw: ctx))
    monkeypatch.setattr(model, "Master", lambda m: SimpleNamespace(generate_text=lambda p, n: {"tokens": [4], "tok_s": 12.5}))
    monkeypatch.setattr(model, "PagedSessions", lambda *a: SimpleNamespace(generate=lambda p, n: {r: [4] for r in p}, tok_s=37.25))
    assert run.main([str(tmp_path), "--prompt-ids", "1,2"]) == 0
    assert capsys.readouterr().out.splitlines() == ["tokens: 4", "tok/s: 12.50"]
    assert run.main([str(tmp_path), "--prompt-ids", "1,2;3"]) == 0
    assert capsys.readouterr().out.splitlines() == ["tokens: 4", "tokens: 4", "tok/s: 37.25"]

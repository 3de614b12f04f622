"""The decoder with an INT8 key/value cache in use over a long time: what passes leave behind, and which recorded steps stay."""
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sgq():
    from __graft_entry__ import load_package
    return load_package()


def decoder(sgq, B, **kw):
    nl = importlib.import_module("sgq_b200.nanollama")
    cfg = nl.NanoLlamaConfig(dim=256, n_layers=2, n_heads=4, hidden=512, vocab=512, max_seq=kw.pop("max_seq", 64))
    return cfg, nl.NanoLlamaInt4(cfg, "cuda", B, seed=3, kv_cache="int8", **kw)


def test_prefixes_and_prompts_leave_no_memory_behind(sgq):
    """A server changes its system prompt and takes prompts of all lengths: once the scratch is as large as it gets, nothing grows."""
    cfg, model = decoder(sgq, 3, max_prefix=500)
    r = np.random.default_rng(1)
    tokens = lambda *s: torch.from_numpy(r.integers(0, cfg.vocab, s))  # noqa: E731
    for n, T in ((500, 60), (63, 21), (32, 5)):                  # the linears' scratch only grows; these sizes take the most of it
        model.set_prefix(tokens(n))
        model.generate(tokens(3, T), 4)
    torch.cuda.synchronize()
    before, step = torch.cuda.memory_allocated(), model._graph
    for n in (1, 2, 3, 17, 100, 250, 333, 400):
        model.set_prefix(tokens(n))
        model.generate(tokens(3, 1 + n % 57), 4)
    torch.cuda.synchronize()
    assert abs(torch.cuda.memory_allocated() - before) < 2 ** 16             # (the allocator's blocks may be a little larger than asked for)
    assert model._graph is step


def test_passes_of_other_sizes_leave_a_recorded_step_alone(sgq):
    """Prompt and prefix passes whose row counts meet the batch, or not, between replays of one recorded step."""
    cfg, model = decoder(sgq, 3, max_prefix=40)
    r = np.random.default_rng(2)
    tokens = lambda *s: torch.from_numpy(r.integers(0, cfg.vocab, s))  # noqa: E731
    prompts = [tokens(3, n) for n in (1, 2, 9)]
    for n in (40, 3, 1, 0, 7):
        prefix = tokens(n)
        want = []
        for p in prompts:
            model.set_prefix(prefix)
            want.append(model.generate(p, 6, use_graph=False, keep_logits=True)[0])
        for p, w in zip(prompts, want):
            model.set_prefix(prefix)
            assert torch.equal(model.generate(p, 6), w)


def test_a_step_is_recorded_again_when_the_scratch_has_grown_and_only_then(sgq):
    """Batches whose linears use the scratch buffer.  Nothing but the model itself touches what generate goes by."""
    cfg, model = decoder(sgq, 20, max_prefix=600)
    r = np.random.default_rng(4)
    tokens = lambda *s: torch.from_numpy(r.integers(0, cfg.vocab, s))  # noqa: E731
    prompt = tokens(20, 1)
    model.generate(prompt, 4)
    step, scratch = model._graph, model.ws.buf
    assert step is not None and model._graph_ws is scratch
    model.set_prefix(tokens(5))
    model.generate(prompt, 4)
    assert model.ws.buf is scratch, "so short a prefix makes the scratch grow: choose a shorter one"
    assert model._graph is step and model._graph_ws is scratch
    model.set_prefix(tokens(600))
    assert model.ws.buf is not scratch, "the prefix does not make the scratch grow: choose a longer one"
    assert model._graph is step and model._graph_ws is scratch           # kept alive as long as the step is
    want, _ = model.generate(prompt, 9, use_graph=False, keep_logits=True)
    assert model._graph is step
    assert torch.equal(model.generate(prompt, 9), want)
    assert model._graph is not step and model._graph_ws is model.ws.buf
    step = model._graph
    assert torch.equal(model.generate(prompt, 9), want) and model._graph is step

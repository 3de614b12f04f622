"""The decoder with an INT8 key/value cache (nanollama.py, kv_cache="int8"): the four cache operators run together as a prompt
pass, decode steps and a shared prefix, against a full recompute in 64 bits that takes the keys and values as they are held."""
import importlib

import numpy as np
import pytest
import torch

from oracle import nanollama_oracle as no
from util import TOL_BF16, TOL_FP32, norm_err

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sgq():
    from __graft_entry__ import load_package
    return load_package()


@pytest.fixture(scope="module")
def nl(sgq):
    return importlib.import_module("sgq_b200.nanollama")


def build(nl, port, B, n_heads, *, seed=3, max_seq=64, **kw):
    cfg = nl.NanoLlamaConfig(dim=256, n_layers=2, n_heads=n_heads, hidden=512, vocab=512, max_seq=max_seq)
    r = np.random.default_rng(seed)
    floats = {}

    def init(name, layer):
        out_f, in_f = nl.weight_shape(cfg, name)
        std = 1.0 if name == "embed" else 2.5 * (2.0 / (in_f + out_f)) ** 0.5
        floats[(name, layer)] = (r.standard_normal((out_f, in_f)) * std).astype(np.float32)
        return torch.from_numpy(floats[(name, layer)])

    model = nl.NanoLlamaInt4(cfg, "cuda", B, init=init, kv_cache="int8", **kw)

    def deq(name, layer):
        w = floats[(name, layer)]
        return port.dequantize_int4(*port.quantize_int4(w, 32), w.shape, 32)

    params = {"embed": floats[("embed", -1)], "n_heads": n_heads, "eps": cfg.eps, "final_norm": np.ones(cfg.dim), "lm_head": deq("lm_head", -1),
              "layers": [{n: deq(n, li) for n in nl.LAYER_WEIGHTS} for li in range(cfg.n_layers)]}
    return cfg, model, params


def held_rows(model, li, P, T):
    """Keys and values of layer li as the model holds them, the prefix in front: [B, h, P + T, hd] in 64 bits, and the scales."""
    out = []
    for which in "kv":
        parts = []
        for cache, n in ((model.prefix_kv[li] if P else None, P), (model.kv[li], T)):
            if cache is not None:
                codes = getattr(cache, which + "_codes")[:, :, :n].cpu().numpy().astype(np.float64)
                scales = getattr(cache, which + "_scales")[:, :, :n].cpu().numpy().astype(np.float64)
                shape = (model.batch,) + codes.shape[1:]
                parts.append((np.broadcast_to(codes, shape), np.broadcast_to(scales, shape[:3])))
        codes, scales = (np.concatenate([p[i] for p in parts], 2) for i in range(2))
        out += [codes * scales[..., None], scales]
    return out


def recompute(params, tokens, rows, tol):
    """forward_full of the oracle with the held keys and values in place of its own, which have to lie within half a step of them
    (and the pass's own tolerance, of the layer's largest value)."""
    B, T = tokens.shape
    H = params["n_heads"]
    h = np.asarray(params["embed"], np.float64)[tokens]
    dim = h.shape[-1]
    hd = dim // H
    cos, sin = no.rope_tables(hd, T)
    at = np.arange(T)
    lin = lambda x, w: x @ np.asarray(w, np.float64).T  # noqa: E731
    heads = lambda x: x.reshape(B, T, H, hd).transpose(0, 2, 1, 3)  # noqa: E731
    one = np.ones(dim)
    for L, (k, ks, v, vs) in zip(params["layers"], rows):
        n = no.rms_norm(h, one)
        q = no.rope(heads(lin(n, L["wq"])), cos, sin, at)
        for own, held, scale in ((no.rope(heads(lin(n, L["wk"])), cos, sin, at), k, ks), (heads(lin(n, L["wv"])), v, vs)):
            assert (np.abs(own - held) <= 0.5 * scale[..., None] * (1 + 2.0 ** -20) + tol * np.abs(own).max()).all()
        a = no.causal_attention(q, k, v)
        h = h + lin(a.transpose(0, 2, 1, 3).reshape(B, T, dim), L["wo"])
        n = no.rms_norm(h, one)
        h = h + lin(no.silu(lin(n, L["w_gate"])) * lin(n, L["w_up"]), L["w_down"])
    return lin(no.rms_norm(h, one), params["lm_head"])


@pytest.mark.parametrize("B,n_heads,P,max_prefix,T,prefill,tol", [
    (2, 2, 0, 0, 9, "simt", TOL_FP32), (3, 4, 0, 0, 1, "simt", TOL_FP32), (2, 4, 37, 40, 9, "simt", TOL_FP32), (3, 2, 1, 130, 1, "simt", TOL_FP32),
    (2, 2, 0, 16, 5, "simt", TOL_FP32), (40, 2, 130, 130, 4, "simt", TOL_FP32), (2, 2, 70, 70, 40, "tc_bf16", 4 * TOL_BF16)])
def test_generation_is_a_full_recompute_over_the_held_rows(sgq, nl, port, B, n_heads, P, max_prefix, T, prefill, tol):
    cfg, model, params = build(nl, port, B, n_heads, max_prefix=max_prefix,
                               prefill_path={"simt": sgq.PATH_SIMT, "tc_bf16": sgq.PATH_TC_BF16}[prefill])
    r = np.random.default_rng(B + P + T)
    n_new = 6
    prefix, prompt = torch.from_numpy(r.integers(0, cfg.vocab, P)), torch.from_numpy(r.integers(0, cfg.vocab, (B, T)))
    if P:
        model.set_prefix(prefix)
    tokens, logits = model.generate(prompt, n_new, use_graph=False, keep_logits=True)
    tokens = tokens.cpu().numpy()
    fed = np.concatenate([np.broadcast_to(prefix.numpy(), (B, P)), prompt.numpy(), tokens[:, :-1]], 1)      # what the caches hold
    want = recompute(params, fed, [held_rows(model, li, P, T + n_new - 1) for li in range(cfg.n_layers)], tol)
    for s in range(n_new):
        assert norm_err(logits[s].cpu().numpy(), want[:, P + T - 1 + s]) <= tol, f"step {s}"
    assert sgq.device_status() == 0


@pytest.mark.parametrize("max_seq", [64, 16000])               # caches for a kernel per head, and dealt out to all warps
@pytest.mark.parametrize("max_prefix", [0, 70])
def test_recorded_steps_are_the_eager_ones(sgq, nl, port, max_prefix, max_seq):
    """One recorded step serves prompts behind every prefix that the model holds in turn."""
    cfg, model, _ = build(nl, port, 3, 4, max_prefix=max_prefix, prefill_path=sgq.PATH_SIMT, max_seq=max_seq)
    r = np.random.default_rng(7)
    prefixes = [torch.from_numpy(r.integers(0, cfg.vocab, n)) for n in (33, 70, 1)] + [None] if max_prefix else [None]
    seen = []
    for prefix in prefixes:
        if max_prefix:
            model.set_prefix(prefix)
        for T in (5, 17):
            prompt = torch.from_numpy(r.integers(0, cfg.vocab, (3, T)))
            want, logits = model.generate(prompt, 9, use_graph=False, keep_logits=True)
            assert torch.equal(model.generate(prompt, 9), want)
            assert model._graph is not None
            seen.append(logits[0])
    assert not any(torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])
    if not max_prefix:
        with pytest.raises(ValueError):
            model.set_prefix(torch.zeros(3, dtype=torch.int64))
    else:
        for bad in (torch.zeros(71, dtype=torch.int64), torch.zeros(1, 3, dtype=torch.int64)):
            with pytest.raises(ValueError):
                model.set_prefix(bad)


def test_recorded_steps_leave_given_back_scratch_alone(sgq, nl, port):
    """Batches whose linears use the scratch buffer: a long prefix makes it grow after a step has been recorded."""
    cfg, model, _ = build(nl, port, 20, 4, max_prefix=600)
    r = np.random.default_rng(8)
    prompt, prefix = torch.from_numpy(r.integers(0, cfg.vocab, (20, 1))), torch.from_numpy(r.integers(0, cfg.vocab, 600))
    model.generate(prompt, 4)
    assert model._graph is not None
    before, at, size = model._graph_ws, model.ws.buf.data_ptr(), model.ws.buf.numel()
    assert before is model.ws.buf
    del before
    model.set_prefix(prefix)
    assert model.ws.buf.numel() > size, "the prefix does not make the scratch grow: choose a longer one"
    want, _ = model.generate(prompt, 9, use_graph=False, keep_logits=True)
    model._graph_ws = None                     # what held the old scratch
    spies = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(4)]
    assert torch.equal(model.generate(prompt, 9), want)
    assert not any(bool(x.any()) for x in spies)
    assert model._graph_ws is model.ws.buf and any(x.data_ptr() == at for x in spies)


def test_a_prefix_in_front_is_the_same_tokens_in_the_prompt(sgq, nl, port):
    """The prefix's tokens once in front or in every prompt: the same definition, so every row that is held is equal up to single
    codes that fp32 noise tips over, and the logits within the fp32 tolerance of their own recompute (above); here the caches."""
    cfg, model, _ = build(nl, port, 2, 2, max_prefix=40, prefill_path=sgq.PATH_SIMT)
    r = np.random.default_rng(9)
    prefix, prompt = torch.from_numpy(r.integers(0, cfg.vocab, 31)), torch.from_numpy(r.integers(0, cfg.vocab, (2, 9)))
    model.set_prefix(prefix)
    model.prefill(prompt)
    behind = held_rows(model, 0, 31, 9)
    model.set_prefix(None)
    model.prefill(torch.cat([prefix.expand(2, 31), prompt], 1))
    whole = held_rows(model, 0, 0, 40)
    for i in (0, 2):               # layer 0's rows do not depend on the attention: a step of a code apart at most
        assert (np.abs(behind[i] - whole[i]) <= 1.001 * whole[i + 1][..., None]).all()
        assert (behind[i] == whole[i]).mean() > 0.99

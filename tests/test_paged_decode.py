"""Prompts, chunks and decode steps of a small W4A16 decoder over a paged cache (kv_cache.plan_pages, rotary.norm_rope_cache and
paged_attention behind tandem_amd.model, and the graph runner), against a numpy restatement of the whole forward pass over the
full sequences, rounded to fp16 where the GPU path stores fp16."""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

import test_decode_step as one_token
from oracle import awq_oracle as o
from tandem_amd import decode_graph, model as tmodel
from tandem_amd.kv_cache import PagedKVCache

CFG = dataclasses.replace(one_token.TINY, qk_norm=True, rope_theta=1e4)


# ------------------------------------------------------------------------------------------- CPU
def test_config_of_the_attention():
    hf = {"hidden_size": 4096, "intermediate_size": 14336, "num_attention_heads": 32, "num_key_value_heads": 8,
          "num_hidden_layers": 32, "vocab_size": 128256, "rms_norm_eps": 1e-5, "model_type": "llama", "rope_theta": 500000.0}
    cfg = tmodel.DecoderConfig.from_hf(hf)
    assert (cfg.head_dim, cfg.qk_norm, cfg.rope_theta, cfg.rope_type) == (128, False, 5e5, "default")
    assert tmodel.DecoderConfig.from_hf({**hf, "rope_theta": None}).rope_theta == 1e4
    assert tmodel.DecoderConfig.from_hf({**hf, "model_type": "qwen3"}).qk_norm
    scaled = tmodel.DecoderConfig.from_hf({**hf, "rope_scaling": {"rope_type": "llama3", "factor": 8.0}})
    assert scaled.rope_type == "llama3"
    with pytest.raises(NotImplementedError, match="llama3"):
        PagedKVCache.for_model(scaled, 4, 1, 64, device="cpu")
    newer = {k: v for k, v in hf.items() if k != "rope_theta"}
    cfg = tmodel.DecoderConfig.from_hf({**newer, "rope_parameters": {"rope_type": "default", "rope_theta": 7e5}})
    assert (cfg.rope_theta, cfg.rope_type) == (7e5, "default")


def test_head_norms_are_parameters_of_qwen3_only():
    with torch.device("meta"):
        names = {n for n, _ in tmodel.DecoderModel(CFG, one_token.AWQ).named_parameters()}
        plain = {n for n, _ in tmodel.DecoderModel(one_token.TINY, one_token.AWQ).named_parameters()}
    heads = {f"model.layers.{i}.self_attn.{x}_norm.weight" for i in range(CFG.num_layers) for x in "qk"}
    assert names - plain == heads


def test_random_weights_are_those_without_head_norms():
    small = dataclasses.replace(CFG, vocab_size=64, num_layers=1)
    got, want = (tmodel.init_random(tmodel.DecoderModel(c), seed=3).state_dict() for c in (small, dataclasses.replace(small, qk_norm=False)))
    assert all(torch.equal(got[n], w) for n, w in want.items())


# ------------------------------------------------------------------------------- helpers
def _model(monkeypatch, seed, cfg=CFG):
    monkeypatch.setattr(one_token, "TINY", cfg)
    m, w = one_token._tiny_model(seed)
    rng = np.random.default_rng(seed + 50)
    for layer, lw in zip(m.model.layers, w["layers"]):
        for name, mod in (("qn", layer.self_attn.q_norm), ("kn", layer.self_attn.k_norm)):
            if mod is not None:
                lw[name] = (0.5 + rng.random(cfg.head_dim)).astype(np.float16)
                mod.weight.copy_(torch.from_numpy(lw[name]))
    return m, w


def _rotate(x, weight, theta, eps):
    """[T, heads, D] float64: norm, rotation by row number, rounded to fp16."""
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    d = x.shape[-1]
    a = np.arange(x.shape[0])[:, None, None] * theta ** (-2.0 * np.arange(d // 2) / d)
    lo, hi = x[..., :d // 2], x[..., d // 2:]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], -1).astype(np.float16).astype(np.float64)


def _oracle(w, ids, cfg=CFG) -> np.ndarray:
    """Logits of every position of one sequence."""
    t, eps, d = len(ids), cfg.rms_norm_eps, cfg.head_dim
    q_size, kv_size, group = cfg.num_heads * d, cfg.num_kv_heads * d, cfg.num_heads // cfg.num_kv_heads
    hidden, residual = w["emb"][np.array(ids)], None
    for lw in w["layers"]:
        if residual is None:
            residual = hidden
            hidden = o.rms_norm(hidden, lw["n1"], eps)
        else:
            hidden, residual = o.add_rms_norm(hidden, residual, lw["n1"], eps)
        qkv = o.linear(hidden, lw["qkv"]).astype(np.float16).astype(np.float64)
        q = _rotate(qkv[:, :q_size].reshape(t, -1, d), lw.get("qn"), cfg.rope_theta, eps)
        k = _rotate(qkv[:, q_size:q_size + kv_size].reshape(t, -1, d), lw.get("kn"), cfg.rope_theta, eps)
        v = qkv[:, q_size + kv_size:].reshape(t, -1, d)
        out = np.empty((t, cfg.num_heads, d))
        for h in range(cfg.num_heads):
            s = q[:, h] @ k[:, h // group].T * d ** -0.5
            s[np.triu_indices(t, 1)] = -np.inf
            p = np.exp(s - s.max(1, keepdims=True))
            out[:, h] = p / p.sum(1, keepdims=True) @ v[:, h // group]
        hidden = o.linear(out.reshape(t, -1).astype(np.float16), lw["o"]).astype(np.float16)
        hidden, residual = o.add_rms_norm(hidden, residual, lw["n2"], eps)
        hidden = o.silu_and_mul(o.linear(hidden, lw["gate_up"])).astype(np.float16)
        hidden = o.linear(hidden, lw["down"]).astype(np.float16)
    hidden, _ = o.add_rms_norm(hidden, residual, w["norm"], eps)
    return o.linear(hidden, w["head"])


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@torch.inference_mode()
def _step(model, cache, tokens, pad=0):
    """One eager step: lane i brings tokens[i]; logits [rows, vocab] of its tokens, lane by lane."""
    new = [len(t) for t in tokens]
    ids = torch.tensor([x for t in tokens for x in t] + [0] * pad, device="cuda")
    batch = cache.plan(_int(new), len(ids), max_query_len=max(new))
    logits = model.compute_logits(model(ids, batch))
    assert batch.counts.tolist() == [sum(new), batch.counts[1].item(), 0, 0]
    return logits[:sum(new)]


# ----------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("qk_norm", [True, False])
def test_prompts_chunks_and_decode_match_oracle(monkeypatch, qk_norm):
    """Ragged prompts in one step, then chunks beside single tokens, padding rows, an idle lane and a reused one."""
    cfg = dataclasses.replace(CFG, qk_norm=qk_norm)
    model, w = _model(monkeypatch, 11, cfg)
    cache = PagedKVCache.for_model(cfg, num_pages=40, max_requests=4, max_seq_len=96)
    cache.keys.fill_(float("nan"))
    cache.values.fill_(float("nan"))
    rng = np.random.default_rng(1)
    seqs = [[], [], [], []]
    plan = [([5, 17, 1, 0], 0), ([1, 1, 1, 30], 2), ([1, 0, 9, 1], 0), ([16, 1, 1, 1], 5), ([1, 1, 1, 1], 0)]
    for i, (new, pad) in enumerate(plan):
        if i == 3:
            cache.release([2])
            seqs[2] = []
        tokens = [rng.integers(0, cfg.vocab_size, n).tolist() for n in new]
        logits = _step(model, cache, tokens, pad)
        at = 0
        for lane, t in enumerate(tokens):
            seqs[lane] += t
            if t:
                want = _oracle(w, seqs[lane], cfg)[-len(t):]
                one_token._close(logits[at:at + len(t)], want, 0.02, (i, lane))
                at += len(t)
    assert cache.context_lens.tolist() == [len(s) for s in seqs]


@pytest.mark.gpu
def test_first_position_is_the_one_token_context(monkeypatch):
    """At position 0 the softmax is over one key: attention over the cache gives the value row, as attend without a batch does."""
    model, _ = _model(monkeypatch, 12)
    ids = [3, 999, 20]
    with torch.inference_mode():
        want = model.compute_logits(model(torch.tensor(ids, device="cuda")))
    cache = PagedKVCache.for_model(CFG, num_pages=8, max_requests=3, max_seq_len=32)
    assert torch.equal(_step(model, cache, [[i] for i in ids]), want)


@pytest.mark.gpu
def test_graph_runner_decodes_over_the_cache(monkeypatch):
    """Replays with idle lanes, padding, releases and eager steps between them equal eager steps over a cache of their own, bit for
    bit, and the oracle; capture leaves the cache as it was."""
    model, w = _model(monkeypatch, 13)
    caches = [PagedKVCache.for_model(CFG, num_pages=30, max_requests=5, max_seq_len=80) for _ in range(2)]
    rng = np.random.default_rng(2)
    seqs = [rng.integers(0, CFG.vocab_size, n).tolist() for n in (4, 33, 1, 15, 16)]
    for c in caches:
        _step(model, c, seqs)
    state = lambda c: [t.clone() for t in (c.context_lens, c.page_table, c.taken, c.keys.view(torch.int16), c.values.view(torch.int16))]  # noqa: E731
    before = state(caches[0])
    runner = decode_graph.DecodeGraphRunner(model, max_bs=5, device=torch.device("cuda", 0), cache=caches[0])
    assert all(torch.equal(a, b) for a, b in zip(before, state(caches[0])))
    for step in range(12):
        lanes = 5 if step % 3 else 3
        ids = rng.integers(0, CFG.vocab_size, lanes).tolist()
        if step % 4 == 1:
            ids[1] = -1
        got = runner.run(ids).clone()
        bs = runner.bucket(lanes)
        tokens = [[i] if i >= 0 else [] for i in ids] + [[] for _ in range(bs - lanes)]
        rows = sum(len(t) for t in tokens)
        want = _step(model, caches[1], tokens, pad=bs - rows)
        assert torch.equal(got, want), step
        at = 0
        for lane, t in enumerate(tokens):
            seqs[lane] += t
            if t:
                if step % 5 == 4:
                    one_token._close(got[at:at + 1], _oracle(w, seqs[lane])[-1:], 0.02, (step, lane))
                at += 1
        if step == 6:
            for c in caches:
                c.release([0])
            seqs[0] = []
    before = state(caches[0])
    assert runner.run([-1, -1, -1]).shape[0] == 0
    assert all(torch.equal(a, b) for a, b in zip(before, state(caches[0])))
    with pytest.raises(ValueError, match="lanes"):
        decode_graph.DecodeGraphRunner(model, max_bs=6, device=torch.device("cuda", 0), cache=caches[0])


@pytest.mark.gpu
def test_lanes_past_their_table_or_without_a_page_stay_alone(monkeypatch):
    """A lane that outgrows its row of the table answers NaN, one that the list has no page for is counted; the others' rows are those of a
    cache with room for all, bit for bit."""
    model, _ = _model(monkeypatch, 15)
    device = torch.device("cuda", 0)
    prompts = [list(range(30)), list(range(9)), list(range(16))]
    rows = []
    for pages, longest in ((30, 64), (30, 32), (5, 32)):
        cache = PagedKVCache.for_model(CFG, num_pages=pages, max_requests=3, max_seq_len=longest)
        _step(model, cache, prompts)  # 2, 1 and 1 pages
        runner = decode_graph.DecodeGraphRunner(model, max_bs=3, device=device, cache=cache)
        rows.append([runner.run([1, 2, -1]).clone() for _ in range(4)])
    for step, (full, narrow, few) in enumerate(zip(*rows)):
        assert torch.equal(narrow[1], full[1]) and torch.equal(few, narrow) if step < 2 else torch.equal(few[1], full[1])
        assert torch.equal(narrow, full) if step < 2 else torch.isnan(narrow[0]).all() and torch.isnan(few[0]).all()
        assert torch.equal(narrow[1], full[1])
    # the last page goes to lane 2; lane 1 fills its page, and then there is none
    for ids, given, lacking in (([-1, 5, 3], 1, 0), ([-1, 5, -1], 0, 0), ([-1, 5, -1], 0, 0), ([-1, 5, 3], 0, 1)):
        got = runner.run(ids)
        assert runner.counts[3].tolist() == [len(got), given, lacking, 0] and torch.isfinite(got).all()
    assert cache.page_table[:, 1].tolist()[1:] == [-1, 4] and int(cache.taken) == 5


@pytest.mark.gpu
def test_two_runners_side_by_side(monkeypatch):
    """Two runners with a cache each, replayed on streams of their own at once, give what one after the other gives."""
    model, _ = _model(monkeypatch, 14)
    device = torch.device("cuda", 0)
    caches = [PagedKVCache.for_model(CFG, num_pages=200, max_requests=2, max_seq_len=2000) for _ in range(3)]
    prompts = [list(range(i, i + 600)) for i in (1, 7)]
    for c in caches:
        _step(model, c, prompts)
    runners = [decode_graph.DecodeGraphRunner(model, max_bs=2, device=device, cache=c) for c in caches]
    want = [runners[2].run([5 + i, 9]).clone() for i in range(6)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for i in range(6):
        for r, st, out in zip(runners, streams, got):
            with torch.cuda.stream(st):
                out.append(r.run([5 + i, 9]).clone())
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.gpu
def test_prompts_in_steps_of_too_few_rows_match_oracle(monkeypatch):
    """Two prompts brought whole to every step of 16 rows: each step computes what fits, and the rest comes again."""
    model, w = _model(monkeypatch, 16)
    cache = PagedKVCache.for_model(CFG, num_pages=20, max_requests=2, max_seq_len=96)
    cache.keys.fill_(float("nan"))
    cache.values.fill_(float("nan"))
    rng = np.random.default_rng(3)
    seqs = [rng.integers(0, CFG.vocab_size, n).tolist() for n in (21, 18)]
    want = [_oracle(w, s) for s in seqs]
    done = [0, 0]
    while done != [21, 18]:
        new = [len(s) - d for s, d in zip(seqs, done)]
        rest = ([x for s, d in zip(seqs, done) for x in s[d:]] + [0] * 16)[:16]
        with torch.inference_mode():
            batch = cache.plan(_int(new), 16)
            starts = batch.query_start.tolist()
            assert starts[-1] == min(sum(new), 16)
            logits = model.compute_logits(model(torch.tensor(rest, device="cuda"), batch))
        for lane, (a, b) in enumerate(zip(starts, starts[1:])):
            if b > a:
                one_token._close(logits[a:b], want[lane][done[lane]:done[lane] + b - a], 0.02, (done, lane))
            done[lane] += b - a
        assert cache.context_lens.tolist() == done


def test_attention_that_the_model_does_not_compute_is_refused():
    """Fields of config.json that ask for another attention than the cache's: at position 0 they do not matter, past it they do."""
    hf = {"hidden_size": 4096, "intermediate_size": 14336, "num_attention_heads": 32, "num_key_value_heads": 8, "num_hidden_layers": 32,
          "vocab_size": 32000, "rms_norm_eps": 1e-5, "model_type": "mistral", "rope_theta": 1e4}
    small = dict(num_pages=2, max_requests=1, device="cpu")
    for change, needle in (({"sliding_window": 4096}, "sliding_window"), ({"partial_rotary_factor": 0.5}, "partial_rotary_factor"),
                           ({"rope_parameters": {"rope_type": "default", "rope_theta": 1e4, "partial_rotary_factor": 0.25}}, "partial_rotary_factor"),
                           ({"attn_logit_softcapping": 50.0}, "attn_logit_softcapping"), ({"attention_bias": True}, "attention_bias"),
                           ({"model_type": "qwen2"}, "attention_bias"), ({"query_pre_attn_scalar": 256}, "query_pre_attn_scalar"),
                           ({"attention_multiplier": 0.5}, "attention_multiplier"),
                           ({"model_type": "qwen3", "sliding_window": 4096, "use_sliding_window": True, "max_window_layers": 8}, "sliding_window"),
                           ({"sliding_window": 4096, "layer_types": ["full_attention"] * 31 + ["sliding_attention"]}, "sliding_window"),
                           ({"layer_types": ["full_attention"] * 31 + ["linear_attention"]}, "layer_types"),
                           ({"rope_parameters": {"full_attention": {"rope_theta": 1e6}, "sliding_attention": {"rope_theta": 1e4}}}, "rope_parameters")):
        cfg = tmodel.DecoderConfig.from_hf({**hf, **change})  # the one-token step takes it as before
        with pytest.raises(NotImplementedError, match=needle):
            PagedKVCache.for_model(cfg, max_seq_len=4097, **small)
    layers = dict(small, max_seq_len=4097)
    for change in ({}, {"sliding_window": None}, {"sliding_window": 5000}, {"sliding_window": 4096, "use_sliding_window": False},
                   {"model_type": "qwen3", "sliding_window": 4096, "use_sliding_window": True, "max_window_layers": 32},
                   {"sliding_window": 4096, "layer_types": ["full_attention"] * 32}, {"attn_logit_softcapping": None},
                   {"partial_rotary_factor": 1.0}, {"query_pre_attn_scalar": 128}, {"attention_bias": False},
                   {"attention_multiplier": 128 ** -0.5}):
        cfg = tmodel.DecoderConfig.from_hf({**hf, **change, "num_hidden_layers": 32})
        PagedKVCache.for_model(dataclasses.replace(cfg, num_layers=1), **layers)
    # a cache that no request can outgrow the window of
    PagedKVCache.for_model(dataclasses.replace(tmodel.DecoderConfig.from_hf({**hf, "sliding_window": 4096}), num_layers=1), **dict(small, max_seq_len=4096))


@pytest.mark.gpu
def test_drafted_tokens_taken_back_match_oracle(monkeypatch):
    """Drafts scored in one pass, most of them taken back, single tokens in the captured step, drafts again: every row is the oracle's for
    the tokens that stayed, and no page is lost."""
    model, w = _model(monkeypatch, 17)
    cache = PagedKVCache.for_model(CFG, num_pages=14, max_requests=2, max_seq_len=112)
    rng = np.random.default_rng(4)
    draw = lambda n: rng.integers(0, CFG.vocab_size, n).tolist()  # noqa: E731
    seqs = [draw(14), draw(30)]
    _step(model, cache, seqs)
    runner = decode_graph.DecodeGraphRunner(model, max_bs=2, device=torch.device("cuda", 0), cache=cache)
    for kept in ((1, 3), (0, 17), (20, 2)):
        drafts = [draw(20), draw(18)]
        logits = _step(model, cache, drafts)
        at = 0
        for lane, (draft, keep) in enumerate(zip(drafts, kept)):
            one_token._close(logits[at:at + len(draft)], _oracle(w, seqs[lane] + draft)[-len(draft):], 0.02, (kept, lane))
            at += len(draft)
            seqs[lane] += draft[:keep]
        cache.context_lens -= _int([20 - kept[0], 18 - kept[1]])
        assert cache.context_lens.tolist() == [len(s) for s in seqs]
        for _ in range(2):
            ids = draw(2)
            got = runner.run(ids).clone()
            for lane, x in enumerate(ids):
                seqs[lane].append(x)
                one_token._close(got[lane:lane + 1], _oracle(w, seqs[lane])[-1:], 0.02, (kept, lane))
        held = [p for r in cache.page_table.tolist() for p in r if p >= 0]
        assert sorted(held + cache.free_pages.tolist()[int(cache.taken):]) == list(range(14))
    cache.release([1, 0])
    assert int(cache.taken) == 0 and sorted(cache.free_pages.tolist()) == list(range(14))

"""One step of speculative decoding through all of its operators: rotary positions, tree attention with shaped scores, the
head's logits, log probabilities, the accepted path, and the append to the cache."""
import threading

import pytest
import torch

from flash_tree_attn_amd import (accept_tree_path, additive_mask_from_parents, append_accepted_kv, apply_rotary, random_tree_parents,
                                 rotary_frequencies, shaped_tree_attention, token_logprobs, tree_depths)
from oracle.kv_append_oracle import append_accepted_kv_oracle
from oracle.step_oracle import accept_path_oracle, logprobs_oracle, rotary_oracle, shaped_attention_oracle

DEV = "cuda"
BSZ, HQ, HKV, L, D, CACHE, VOCAB = 3, 4, 2, 13, 64, 640, 8


class Model:
    """One attention layer and a head over a small vocabulary, so that the drafts of `random_tree_parents` trees hit."""

    def __init__(self, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)
        self.embedding, self.wq, self.wk, self.wv = r(VOCAB, 64), r(64, HQ * D) / 8, r(64, HKV * D) / 8, r(64, HKV * D) / 8
        self.head = r(HQ * D, VOCAB) / 4
        self.k_cache, self.v_cache = r(BSZ, HKV, CACHE, D), r(BSZ, HKV, CACHE, D)
        self.inv_freq = rotary_frequencies(D, device=DEV)[0]
        self.slopes = 2.0 ** -torch.arange(1, HQ + 1, device=DEV).float()
        self.opt = dict(softcap=30.0, window=200, slopes=self.slopes, kv_group_num=HQ // HKV)
        parents = [random_tree_parents(L, g) for _ in range(BSZ)]
        self.parents = torch.stack(parents).to(DEV)
        self.mask = torch.stack([additive_mask_from_parents(p) for p in parents])[:, None].to(DEV)
        self.depths = torch.stack([tree_depths(p) for p in parents]).to(DEV)
        self.lens = torch.tensor([600, 64, 0], device=DEV)

    def project(self, tokens):
        x = self.embedding[tokens]
        heads = lambda w, n: (x @ w).view(BSZ, L, n, D).transpose(1, 2)
        return heads(self.wq, HQ), heads(self.wk, HKV), heads(self.wv, HKV)

    def step(self, tokens, new_lens):
        """Everything the step produces, by name; the cache is updated in place, the lengths go to new_lens."""
        s = {}
        s["q0"], s["k0"], v = self.project(tokens)
        s["q"], s["k"] = apply_rotary(s["q0"], s["k0"], self.depths, self.inv_freq, kv_seq_len=self.lens)
        s["v"] = v
        s["out"] = shaped_tree_attention(s["q"], self.k_cache, self.v_cache, s["k"], v, self.mask, self.lens, depths=self.depths, **self.opt)
        s["logits"] = s["out"].transpose(1, 2).reshape(BSZ, L, HQ * D) @ self.head
        s["scores"] = token_logprobs(s["logits"], tokens[..., None], top_k=3, temperature=0.7)
        s["targets"] = s["scores"].top_ids[..., 0]
        s["path"] = accept_tree_path(tokens, self.parents, s["targets"])
        append_accepted_kv(self.k_cache, self.v_cache, s["k"], v, s["path"][0], s["path"][1], self.lens, new_lens)
        return s


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_steps_match_the_definitions(dtype):
    """Each operator against its definition on the inputs that the one before produced, over steps that follow one another.
    Attention's bound: half a step of the type for the result, and of each weight (they move a mean of values up to max |v|
    by as much again), doubled for the 32-bit rest; log probabilities: 32-bit sums of 8 terms."""
    m = Model(dtype, 1)
    half = torch.finfo(dtype).eps / 2
    g = torch.Generator().manual_seed(2)
    accepted = 0
    for _ in range(5):
        tokens = torch.randint(0, VOCAB, (BSZ, L), generator=g).to(DEV)
        before_k, before_v = m.k_cache.clone(), m.v_cache.clone()
        new_lens = torch.empty_like(m.lens)
        s = m.step(tokens, new_lens)
        for got, x in ((s["q"], s["q0"]), (s["k"], s["k0"])):
            want = rotary_oracle(x, m.depths, m.inv_freq, m.lens)
            assert float(((got.double() - want).abs() - half * want.abs()).max()) < 2e-6
        want = shaped_attention_oracle(s["q"], before_k, before_v, s["k"], s["v"], m.mask, m.lens, depths=m.depths,
                                       **{n: v for n, v in m.opt.items() if n != "kv_group_num"})
        vmax = float(max(before_v.abs().max(), s["v"].abs().max()))
        assert float(((s["out"].double() - want).abs() - 2 * half * (want.abs() + 2 * vmax)).max()) < 1e-4
        logp, entropy, lse, top, ids = logprobs_oracle(s["logits"], tokens[..., None], 3, 0.7)
        for got, want in ((s["scores"].logprobs, logp), (s["scores"].entropy, entropy), (s["scores"].lse, lse), (s["scores"].top_logprobs, top)):
            torch.testing.assert_close(got.double(), want, atol=2e-5, rtol=2e-6)
        assert torch.equal(s["scores"].top_ids, ids)
        for got, want in zip(s["path"], accept_path_oracle(tokens.cpu(), m.parents.cpu(), s["targets"].cpu())):
            assert torch.equal(got.cpu(), want)
        k_want, v_want, n_want = (t.to(DEV) for t in append_accepted_kv_oracle(before_k, before_v, s["k"], s["v"], *s["path"][:2], m.lens))
        assert torch.equal(m.k_cache, k_want) and torch.equal(m.v_cache, v_want) and torch.equal(new_lens, n_want)
        accepted += int(s["path"][1].sum())
        m.lens = new_lens
    assert accepted > 5 * BSZ        # not the roots alone


@pytest.mark.gpu
def test_two_captured_steps_replay_what_eager_steps_give():
    """Two steps of different models in two graphs, replayed in turn with eager work between: every replay gives what the
    eager step gave (the graphs have workspaces of their own; nothing is left over from one replay to the next)."""
    sides, inputs = [], []
    g = torch.Generator().manual_seed(3)
    for seed in (4, 5):
        m = Model(torch.bfloat16, seed)
        tokens = torch.randint(0, VOCAB, (BSZ, L), generator=g).to(DEV)
        cache = m.k_cache.clone(), m.v_cache.clone()
        eager_lens, lens = torch.empty_like(m.lens), torch.empty_like(m.lens)
        eager = m.step(tokens, eager_lens)
        after = m.k_cache.clone(), m.v_cache.clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            s = m.step(tokens, lens)
        sides.append((m, cache, eager, after, eager_lens, graph, s, lens))
        inputs.append(tokens)     # the graph reads them at every replay
    for turn in range(3):
        for m, cache, eager, after, eager_lens, graph, s, lens in sides:
            m.k_cache.copy_(cache[0])
            m.v_cache.copy_(cache[1])
            for n in ("out", "q", "k"):
                s[n].fill_(float("nan"))
            lens.zero_()
            graph.replay()
            token_logprobs(torch.randn(64, 70000, device=DEV), top_k=5)     # eager work with a workspace of its own
            torch.cuda.synchronize()
            assert all(torch.equal(s[n], eager[n]) for n in ("q", "k", "out", "logits", "targets")), turn
            assert all(torch.equal(a, b) for a, b in zip(s["scores"], eager["scores"])) and all(torch.equal(a, b) for a, b in zip(s["path"], eager["path"]))
            assert torch.equal(lens, eager_lens) and torch.equal(m.k_cache, after[0]) and torch.equal(m.v_cache, after[1])


@pytest.mark.gpu
def test_threads_with_streams_of_their_own():
    """Four threads at once, each with a model and a stream: every step gives what it gives alone."""
    g = torch.Generator().manual_seed(6)
    tokens = torch.randint(0, VOCAB, (BSZ, L), generator=g).to(DEV)
    models = [Model(torch.float16, 10 + i) for i in range(4)]
    caches = [(m.k_cache.clone(), m.v_cache.clone()) for m in models]
    alone = [m.step(tokens, torch.empty_like(m.lens)) for m in models]
    torch.cuda.synchronize()
    failures = []

    def run(m, cache, want):
        try:
            stream = torch.cuda.Stream()
            with torch.no_grad(), torch.cuda.stream(stream):
                for _ in range(20):
                    m.k_cache.copy_(cache[0])
                    m.v_cache.copy_(cache[1])
                    s = m.step(tokens, torch.empty_like(m.lens))
                    stream.synchronize()
                    assert torch.equal(s["out"], want["out"]) and torch.equal(s["path"][0], want["path"][0])
                    assert all(torch.equal(a, b) for a, b in zip(s["scores"], want["scores"]))
        except Exception as error:
            failures.append(error)

    threads = [threading.Thread(target=run, args=a) for a in zip(models, caches, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[0]

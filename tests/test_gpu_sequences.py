"""A model's layers for sequences side by side: prompts in chunks next to tokens, forks, drafts in a tree, compaction, by the
operators together, against the layers in 64 bits.

Tolerance of all: per layer some 13 tensors are rounded to bf16 (half a step, at most 2^-8 of a value, 2^-9.8 rms), each of a branch
that is at most the sum's size, twice over in the worst case: 2 layers * 13 * 2^-9.8 < 0.03 if all errors added up, 0.006 as
independent ones; 0.02 lies between.
"""

import argparse
import math

import pytest
import torch

import svdmlp
from svdmlp import e2e_block

pytestmark = pytest.mark.gpu
H, I, R, HEADS, KV, LAYERS, THETA = 512, 1024, 256, 8, 2, 2, 500000.0


def _weights(gpu, seed, head_norms):
    gen = torch.Generator(device=gpu)
    gen.manual_seed(seed)
    weights = [e2e_block.make_layer_weights(gen, gpu, H, I, R, HEADS, KV, torch.bfloat16) for _ in range(LAYERS)]
    if head_norms:
        for w in weights:
            for name in ("q_norm_w", "k_norm_w"):
                w[name] = (1 + 0.2 * torch.randn(H // HEADS, generator=gen, device=gpu)).to(torch.bfloat16)
    return weights, lambda *shape: (torch.randn((*shape, H), generator=gen, device=gpu) * 0.02).to(torch.bfloat16)


def _layers64(x, weights, positions=None, sees=None):
    """The layers over one sequence's rows in 64 bits; sees (T, T): which row sees which."""
    x = x.double().cpu()
    T, D = x.shape[0], H // HEADS
    positions = torch.arange(T) if positions is None else positions
    sees = torch.ones(T, T).tril().bool() if sees is None else sees
    angle = positions.double()[:, None] * THETA ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]

    def norm(t, w):
        return t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w

    def turn(t, gain):
        t = norm(t, gain) if gain is not None else t
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    for w in weights:
        w = {k: v.double().cpu() for k, v in w.items()}
        n = norm(x, w["norm1_w"])
        q, k = turn((n @ w["wq"]).view(T, HEADS, D), w.get("q_norm_w")), turn((n @ w["wk"]).view(T, KV, D), w.get("k_norm_w"))
        k, v = k.repeat_interleave(HEADS // KV, 1), (n @ w["wv"]).view(T, KV, D).repeat_interleave(HEADS // KV, 1)
        s = torch.einsum("thd,uhd->htu", q, k) / math.sqrt(D)
        s = s.masked_fill(~sees, -math.inf).softmax(-1)
        x = x + torch.einsum("htu,uhd->thd", s, v).reshape(T, H) @ w["wo"]
        n = norm(x, w["norm2_w"])
        x = x + (torch.nn.functional.silu(n @ w["ug"] @ w["vg"]) * (n @ w["uu"] @ w["vu"])) @ w["ud"] @ w["vd"]
    return x


def _close(got, want):
    got = got.double().cpu()
    assert got.shape == want.shape and float((got - want).norm() / want.norm()) < 0.02


@pytest.mark.parametrize("head_norms", [False, True])
def test_prompt_in_chunks(gpu, head_norms):
    weights, rows = _weights(gpu, 1, head_norms)
    x = rows(150)
    want = _layers64(x, weights)
    model = e2e_block.DecoderModel(weights, HEADS, KV, 150)
    for a, z in ((0, 70), (70, 71), (71, 71), (71, 150)):
        _close(model.extend(x[a:z], a), want[a:z]) if z > a else model.extend(x[a:z], a)
    _close(model.step(x[149:], 149), want[149:])
    _close(e2e_block.DecoderModel(weights, HEADS, KV, 150).prompt(x), want)
    with pytest.raises(ValueError, match="positions"):
        model.extend(x[:2], 191)
    with pytest.raises(ValueError, match="positions"):
        model.extend(x[:2], -1)


@pytest.mark.parametrize("head_norms", [False, True])
def test_sequences_side_by_side(gpu, head_norms):
    """Two prompts in chunks next to each other's tokens, a fork, drafts in a tree of which some stay, a compaction, and on."""
    weights, rows = _weights(gpu, 2, head_norms)
    model = e2e_block.SequenceModel(weights, HEADS, KV, 12, THETA)
    pool, told = model.pool, {}

    def step(sequences, tokens):
        x = rows(sum(tokens))
        got, at = model.step(x, sequences, tokens), 0
        for s, t in zip(sequences, tokens):
            told[s] = torch.cat([told.get(s, x[:0]), x[at:at + t]])
            if t:
                _close(got[at:at + t], _layers64(told[s], weights)[-t:])
            at += t

    a, b = pool.add(), pool.add()
    step([a], [100])
    step([b, a], [37, 1])
    step([a, b], [1, 90])
    c = pool.fork(a)
    told[c] = told[a]
    step([c, b, a], [3, 1, 1])
    step([a, b, c], [1, 0, 1])
    # five drafts each: 0 - 1 - 2, and 0 - 3 - 4
    tree = torch.tensor([[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 1, 1, 0, 0], [1, 0, 0, 1, 0], [1, 0, 0, 1, 1]]).bool()
    x = rows(2, 5)
    got = model.verify(x, [a, c], tree.to(gpu))
    for i, s in enumerate((a, c)):
        n = told[s].shape[0]
        sees = torch.ones(n + 5, n + 5).tril().bool()
        sees[n:, n:] = tree
        positions = torch.cat([torch.arange(n), n + tree.sum(1) - 1])
        _close(got[i], _layers64(torch.cat([told[s], x[i]]), weights, positions, sees)[n:])
    d = pool.fork(a)
    with pytest.raises(ValueError, match="fork"):
        model.keep([a, c], [[0, 3, 4], []], 5)
    pool.free(d)
    model.keep([a, c], [[0, 3, 4], []], 5)
    told[a] = torch.cat([told[a], x[0, [0, 3, 4]]])
    assert pool.length(a) == told[a].shape[0] and pool.length(c) == told[c].shape[0]
    step([c, a], [1, 1])
    pool.free(b)
    assert pool.compact() == 12 - pool.free_pages
    step([a, c], [1, 70])
    with pytest.raises(ValueError, match="tokens"):
        model.step(rows(3), [a, c], [1, 1])
    with pytest.raises(ValueError, match="once"):
        model.step(rows(2), [a, a], [1, 1])
    with pytest.raises(ValueError, match="increasing"):
        model.keep([a], [[1, 0]], 5)
    held = pool.length(a), pool.length(c), pool.free_pages
    for x, t in ((rows(2, 3), tree.to(gpu)), (rows(2, 5), tree), (rows(2, 5), tree.to(gpu).int()), (rows(1, 5), tree.to(gpu)), (rows(2, 0), tree[:0, :0].to(gpu))):
        with pytest.raises(ValueError, match="tree"):
            model.verify(x, [a, c], t)
    with pytest.raises(ValueError, match="once"):
        model.keep([a, a], [[0], [1]], 5)
    with pytest.raises(ValueError, match="fewer"):
        model.keep([pool.add()], [[0]], 5)
    assert held == (pool.length(a), pool.length(c), pool.free_pages)


def test_books_of_a_captured_stream(gpu):
    pool = svdmlp.PagePool(torch.zeros(2, 3, 4, 1, 8, device=gpu))
    a = pool.add()
    torch.cuda.synchronize()
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device=gpu)
    with torch.cuda.graph(graph):
        x.add_(1)
        for call in (lambda: pool.reserve([a], [1]), lambda: pool.table([a]), pool.compact):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    assert pool.length(a) == 0 and pool.free_pages == 3


def test_extend_captured(gpu):
    """A chunk as one graph, replayed after its caches and rows changed."""
    weights, rows = _weights(gpu, 3, True)
    model = e2e_block.DecoderModel(weights, HEADS, KV, 128)
    x = rows(100)
    model.extend(x[:60], 0)
    inp = x[60:].clone()
    model.extend(inp, 60)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.extend(inp, 60)
    for seed in range(3):
        other = x.roll(seed + 1, 0)
        model.extend(other[:60], 0)
        inp.copy_(other[60:])
        want = model.extend(inp, 60).clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("head_norms", [False, True])
def test_e2e_record_of_the_serve_arm(gpu, head_norms):
    args = argparse.Namespace(layers=2, model_path=None, compress_ratio=0.8, warmup=1, repeats=2, seed=3, dense_arm=False, serve_arm=True,
                              serve_sequences=3, serve_chunk=40)
    rec = e2e_block.bench_model(70, dict(hidden=H, intermediate=I, heads=HEADS, kv_heads=KV, layers=2, head_norms=head_norms), args)
    served = rec["served_step"]
    assert served["chunks_vs_prompt_relative_l2"] < 0.02 and served["iterations"] == 2 and 0 < served["latency_ms_min"]
    args.serve_chunk = 0
    with pytest.raises(ValueError, match="serve-chunk"):
        e2e_block.bench_model(70, dict(hidden=H, intermediate=I, heads=HEADS, kv_heads=KV, layers=2), args)

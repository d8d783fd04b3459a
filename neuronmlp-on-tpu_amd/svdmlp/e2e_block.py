"""Whole-model N-layer transformer prefill: fused SVD MLP vs unfused SVD MLP
(bench/e2e_block.py:1-439), on MI355X.

Every layer is RMSNorm -> GQA attention -> residual -> RMSNorm -> MLP ->
residual (bench/e2e_block.py:229-278), with RMSNorm eps 1e-6 and the
reference's synthetic weights (unit norm gains, N(0, 1/fan_in) projections,
X ~ 0.02 N(0, 1)).  The arms differ only in how the SVD MLP runs:

* ``fused_block``: the library's block entry point ``ops.svd_mlp_block``
  (RMSNorm, the fused SVD-MLP layer and the residual add, all HIP kernels);
* ``unfused_block``: RMSNorm and six plain GEMMs with an fp32 SiLU
  (``compat._unfused_low_rank_pallas``, the reference's
  ``nki_matmul_fully_optimized_`` arm, on the vendor library);
* ``dense_block`` (``--dense-arm``, not in the reference's report): the
  dense SwiGLU (``compat.nki_baseline``) on weights rebuilt as U.V.
* ``decoder_block`` and ``decoder_step`` (``--decoder-arm``, not in the
  reference's report): the layers as a served model runs them, causal and with
  rotary positions, all but the projections in the library's kernels
  (:mod:`svdmlp.decoder`): a prompt of S tokens that fills a paged cache, and
  one more token onto it.
* ``served_step`` (``--serve-arm``, not in the reference's report): a step of the
  same layers for several sequences (:class:`SequenceModel`), the first prompts read
  in chunks: each generates a token onto S, and one reads a chunk of its prompt.

Attention is the same in the other arms and is not the subject of the comparison:
torch's scaled_dot_product_attention, restricted to its flash and
memory-efficient kernels (non-causal, as ``jax.nn.dot_product_attention`` is
called at bench/e2e_block.py:222), with the KV heads repeated per group.
Times are hipEvent-timed whole-model forward passes; the report keeps the
reference's keys (bench/e2e_block.py:338-352, 399-413).

    python -m svdmlp.e2e_block --model llama3-8b --seq-lens 128 512 1024 --layers 4
"""

from __future__ import annotations

import argparse
import contextlib
import json
import math
import statistics
import sys

_SHAPES = {
    "llama3-3b": dict(hidden=3072, intermediate=8192, heads=24, kv_heads=8, layers=28),
    "llama3-8b": dict(hidden=4096, intermediate=14336, heads=32, kv_heads=8, layers=32),
    # queries and keys normalised head by head (by the decoder and the server only)
    "qwen3-8b": dict(hidden=4096, intermediate=12288, heads=32, kv_heads=8, layers=36, head_norms=True),
}
_DEFAULT_COMPRESS_RATIO = 0.8
RMS_EPS = 1e-6
_WEIGHT_KEYS = ("norm1_w", "norm2_w", "wq", "wk", "wv", "wo", "ug", "vg", "uu", "vu", "ud", "vd")


def rmsnorm(x, w, eps: float = RMS_EPS):
    """bench/e2e_block.py:72-75: fp32 x / sqrt(mean(x^2) + eps) * w, cast back."""
    import torch

    x32 = x.float()
    rms = torch.sqrt(torch.mean(x32 * x32, dim=-1, keepdim=True) + eps)
    return (x32 / rms * w.float()).to(x.dtype)


def attention(x, wq, wk, wv, wo, num_heads: int, num_kv_heads: int):
    """Grouped-query attention over one sequence (bench/e2e_block.py:205-226):
    q, k, v projections, KV heads repeated per group, non-causal softmax
    attention with scale 1/sqrt(head_dim), output projection."""
    import torch
    from torch.nn.attention import SDPBackend, sdpa_kernel

    S, H = x.shape
    head_dim = H // num_heads
    groups = num_heads // num_kv_heads
    q = (x @ wq).view(S, num_heads, head_dim).transpose(0, 1)
    k = (x @ wk).view(S, num_kv_heads, head_dim).transpose(0, 1).repeat_interleave(groups, dim=0)
    v = (x @ wv).view(S, num_kv_heads, head_dim).transpose(0, 1).repeat_interleave(groups, dim=0)
    if x.device.type == "cuda":
        # flash / memory-efficient kernels only: the math fallback runs batched
        # bf16 products on transposed views
        with sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]):
            out = torch.nn.functional.scaled_dot_product_attention(q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0))[0]
    else:
        scores = (q.float() @ k.float().transpose(-1, -2)) / math.sqrt(head_dim)
        out = (torch.softmax(scores, dim=-1) @ v.float()).to(x.dtype)
    return out.transpose(0, 1).reshape(S, H) @ wo


def make_layer_weights(gen, device, H: int, I: int, R: int, num_heads: int, num_kv_heads: int, dtype):
    """Synthetic weights of one layer (bench/e2e_block.py:88-115): unit norm
    gains, N(0, 1/fan_in) projections and SVD factors, drawn from ``gen``."""
    import torch

    kv_dim = num_kv_heads * (H // num_heads)

    def rand(shape, fan_in):
        return (torch.randn(shape, generator=gen, device=device, dtype=torch.float32) / math.sqrt(fan_in)).to(dtype)

    return dict(
        norm1_w=torch.ones(H, device=device, dtype=dtype), norm2_w=torch.ones(H, device=device, dtype=dtype),
        wq=rand((H, H), H), wk=rand((H, kv_dim), H), wv=rand((H, kv_dim), H), wo=rand((H, H), H),
        ug=rand((H, R), H), vg=rand((R, I), R), uu=rand((H, R), H), vu=rand((R, I), R),
        ud=rand((I, R), I), vd=rand((R, H), R))


def load_checkpoint_weights(model_path, layer_indices, device, dtype):
    """Real weights of the selected layers (bench/e2e_block.py:118-197):
    attention projections and norm gains straight from the safetensors
    shards (2-D Linear weights transposed to (in, out)), MLP factors through
    :func:`svdmlp.checkpoint.load_mlp_factors`."""
    from contextlib import ExitStack
    from pathlib import Path

    from safetensors import safe_open

    from . import checkpoint

    model_path = Path(model_path)
    _, index = checkpoint.checkpoint_metadata(model_path)
    weight_map = index["weight_map"]
    attn = ("self_attn.q_proj.weight", "self_attn.k_proj.weight", "self_attn.v_proj.weight",
            "self_attn.o_proj.weight", "input_layernorm.weight", "post_attention_layernorm.weight")
    keys = [f"model.layers.{layer}.{suffix}" for layer in layer_indices for suffix in attn]
    missing = [k for k in keys if k not in weight_map]
    if missing:
        raise KeyError(f"checkpoint missing key: {missing[0]}")
    norms = ("self_attn.q_norm.weight", "self_attn.k_norm.weight")  # of models that have them
    keys += [k for layer in layer_indices for k in (f"model.layers.{layer}.{n}" for n in norms) if k in weight_map]
    raw = {}
    with ExitStack() as stack:
        shards = {name: stack.enter_context(safe_open(str(model_path / name), framework="pt"))
                  for name in sorted({weight_map[k] for k in keys})}
        for k in keys:
            t = shards[weight_map[k]].get_tensor(k)
            raw[k] = (t.t() if t.dim() == 2 else t).contiguous().to(device=device, dtype=dtype)
    factors = checkpoint.load_mlp_factors(model_path, layer_indices, device=device, dtype=dtype)
    out = []
    for layer, (ug, vg, uu, vu, ud, vd) in zip(layer_indices, factors):
        p = f"model.layers.{layer}."
        out.append(dict(norm1_w=raw[p + "input_layernorm.weight"], norm2_w=raw[p + "post_attention_layernorm.weight"],
                        wq=raw[p + "self_attn.q_proj.weight"], wk=raw[p + "self_attn.k_proj.weight"],
                        wv=raw[p + "self_attn.v_proj.weight"], wo=raw[p + "self_attn.o_proj.weight"],
                        ug=ug, vg=vg, uu=uu, vu=vu, ud=ud, vd=vd))
        if p + norms[0] in raw and p + norms[1] in raw:
            out[-1].update(q_norm_w=raw[p + norms[0]], k_norm_w=raw[p + norms[1]])
    return out


def unfused_block(x, w, num_heads: int, num_kv_heads: int):
    """bench/e2e_block.py:229-253: attention, then six plain GEMMs."""
    from . import compat

    x = x + attention(rmsnorm(x, w["norm1_w"]), w["wq"], w["wk"], w["wv"], w["wo"], num_heads, num_kv_heads)
    h = rmsnorm(x, w["norm2_w"])
    return x + compat._unfused_low_rank_pallas(h, w["uu"], w["vu"], w["ug"], w["vg"], w["ud"], w["vd"])


def fused_block(x, w, num_heads: int, num_kv_heads: int, workspace=None):
    """bench/e2e_block.py:256-278: attention, then the library's MLP block
    (RMSNorm, fused SVD MLP and residual in HIP kernels)."""
    from . import ops

    x = x + attention(rmsnorm(x, w["norm1_w"]), w["wq"], w["wk"], w["wv"], w["wo"], num_heads, num_kv_heads)
    return ops.svd_mlp_block(x, w["norm2_w"].float(), w["ug"], w["vg"], w["uu"], w["vu"], w["ud"], w["vd"],
                             eps=RMS_EPS, workspace=workspace)


def dense_block(x, w, dense, num_heads: int, num_kv_heads: int):
    """Dense comparison arm: attention, then the dense SwiGLU
    (test_speedup.py:669-678) on ``dense`` = (up_proj, gate_proj, down_proj)."""
    from . import compat

    x = x + attention(rmsnorm(x, w["norm1_w"]), w["wq"], w["wk"], w["wv"], w["wo"], num_heads, num_kv_heads)
    return x + compat.nki_baseline(rmsnorm(x, w["norm2_w"]), *dense)


class _Layers:
    """The layers of ``weights`` as a served model runs them, on the library's
    kernels: q, k, v from one product, rotary positions (of heads that are normalised
    first where the weights have ``q_norm_w`` and ``k_norm_w``), a paged cache a
    layer, causal attention, the SVD MLP, and each residual sum with the norm after
    it.  ``caches[i]`` (2, pages, PAGE, kv heads, head size): layer i's keys and values."""

    PAGE = 64

    def __init__(self, weights, num_heads: int, num_kv_heads: int, pages: int, theta: float, workspace):
        import torch

        from . import decoder

        self.weights, self.workspace = weights, workspace
        self.heads = (num_heads, num_kv_heads, num_kv_heads)
        H, like = weights[0]["wq"].shape[0], weights[0]["wq"]
        self.head_dim = H // num_heads
        self.qkv = [torch.cat([w["wq"], w["wk"], w["wv"]], dim=1) for w in weights]
        self.gains = [(w["norm1_w"].float(), w["norm2_w"].float()) for w in weights]
        self.head_gains = [(w["q_norm_w"].float(), w["k_norm_w"].float()) if "q_norm_w" in w else None for w in weights]
        self.caches = like.new_zeros((len(weights), 2, pages, self.PAGE, num_kv_heads, self.head_dim))
        self.inv_freq, self.rope_scale = decoder.rope_frequencies(self.head_dim, theta, device=like.device)

    def _layers(self, x, positions, slots, attend):
        from . import decoder, ops

        T = x.shape[0]
        _, n = decoder.residual_norm(x, None, self.gains[0][0], eps=RMS_EPS)
        for i, w in enumerate(self.weights):
            q, k, v = (n @ self.qkv[i]).view(T, -1, self.head_dim).split(self.heads, dim=1)
            keys, values = self.caches[i]
            if self.head_gains[i] is None:
                q = decoder.rope_append(q, k, v, positions, self.inv_freq, keys, values, slots, scale=self.rope_scale)
            else:
                q = decoder.norm_rope_append(q, k, v, positions, self.inv_freq, *self.head_gains[i], keys, values, slots, eps=RMS_EPS,
                                             scale=self.rope_scale)
            x, n = decoder.residual_norm(x, attend(q, keys, values).reshape(T, -1) @ w["wo"], self.gains[i][1], eps=RMS_EPS)
            y = ops.svd_mlp(n, w["ug"], w["vg"], w["uu"], w["vu"], w["ud"], w["vd"], workspace=self.workspace)
            x, n = decoder.residual_norm(x, y, self.gains[i + 1][0] if i + 1 < len(self.weights) else None, eps=RMS_EPS)
        return x


class DecoderModel(_Layers):
    """:class:`_Layers` for one sequence, its pages in order.

    ``prompt(x)`` runs a sequence and fills the caches; ``extend(x, first)`` runs the
    tokens from position ``first`` on, a chunk of a prompt, whose keys and values go
    into the caches, onto what they hold before them; ``step(x, position)`` one token.
    ``capacity``: tokens the caches can hold."""

    def __init__(self, weights, num_heads: int, num_kv_heads: int, capacity: int, theta: float = 500000.0, workspace=None):
        import torch

        pages = -(-capacity // self.PAGE)
        super().__init__(weights, num_heads, num_kv_heads, pages, theta, workspace)
        device = self.caches.device
        # one sequence: its pages lie in order, so a prompt's keys are the cache's first rows
        self.table = torch.arange(pages, dtype=torch.int32, device=device)[None]
        self.places = torch.arange(pages * self.PAGE, device=device)
        self.lengths = torch.arange(pages * self.PAGE + 1, dtype=torch.int32, device=device)

    def prompt(self, x):
        from . import decoder

        rows = x.shape[0]

        def attend(q, keys, values):
            return decoder.prompt_attention(q, keys.flatten(0, 1)[:rows], values.flatten(0, 1)[:rows])

        return self._at(x, 0, attend)

    def extend(self, x, first: int):
        from . import decoder

        rows = x.shape[0]
        if not rows:
            return x
        lengths, cu = self.lengths[first + rows:first + rows + 1], self.lengths[:rows + 1:rows]
        return self._at(x, first, lambda q, keys, values: decoder.chunk_attention(q, keys, values, self.table, lengths, cu))

    def step(self, x, position: int):
        from . import decoder

        lengths = self.lengths[position + 1:position + 2]
        return self._at(x, position, lambda q, keys, values: decoder.cache_attention(q[None], keys, values, self.table, lengths)[0])

    def _at(self, x, first: int, attend):
        T = x.shape[0]
        if first < 0 or first + T > self.places.shape[0]:
            raise ValueError(f"positions {first} to {first + T - 1} of caches for {self.places.shape[0]} tokens")
        at = self.places[first:first + T]
        return self._layers(x, at, at, attend)


class SequenceModel(_Layers):
    """:class:`_Layers` for sequences side by side in caches of ``pages`` pages, whose
    books :class:`svdmlp.PagePool` keeps (``pool``: sequences are added, forked,
    trimmed and freed there).

    ``step(x, sequences, tokens)`` runs the next tokens[i] tokens of sequence
    sequences[i], rows of x in this order: one where it generates, a chunk of its
    prompt where that is being read, in one call.  ``verify(x, sequences, tree)``
    runs a tree of drafts of each, and ``keep(sequences, paths, drafts)`` puts the
    accepted ones behind the context.  A step or a tree that raises leaves the
    sequences as long as they were."""

    def __init__(self, weights, num_heads: int, num_kv_heads: int, pages: int, theta: float = 500000.0, workspace=None):
        from .pages import PagePool

        super().__init__(weights, num_heads, num_kv_heads, pages, theta, workspace)
        self.pool = PagePool(self.caches.flatten(0, 1))

    @contextlib.contextmanager
    def _reserved(self, sequences, tokens):
        """(slots, positions, cu_seqlens, block_table, lengths) of room for tokens[i] more of sequences[i], given back by
        what raises."""
        before = [self.pool.length(s) for s in sequences]
        room = self.pool.reserve(sequences, tokens)
        try:
            yield *room, *self.pool.table(sequences)
        except BaseException:
            for s, length in zip(sequences, before):
                self.pool.trim(s, length)
            raise

    def step(self, x, sequences, tokens):
        from . import decoder

        sequences, tokens = list(sequences), [int(t) for t in tokens]
        if sum(tokens) != x.shape[0]:
            raise ValueError(f"{sum(tokens)} tokens in {x.shape[0]} rows")
        if not sum(tokens):
            return x
        with self._reserved(sequences, tokens) as (slots, positions, cu, table, lengths):
            return self._layers(x, positions, slots, lambda q, keys, values: decoder.chunk_attention(q, keys, values, table, lengths, cu))

    def verify(self, x, sequences, tree):
        """x (sequences, n, hidden): n drafts of each sequence, their states.  tree
        (n, n), bool: whose row i names the drafts that draft i follows, and itself,
        which all come before it.  Those are in the caches until keep says which stay."""
        from . import decoder

        B, n, H = x.shape
        if len(sequences) != B or tuple(tree.shape) != (n, n) or not 1 <= n <= 64:
            raise ValueError(f"{len(sequences)} sequences and a tree {tuple(tree.shape)} for {B} x {n} drafts (1 to 64)")
        if str(tree.dtype) != "torch.bool" or tree.device != x.device:
            raise ValueError(f"the tree must be a bool tensor on {x.device}, got {tree.dtype} on {tree.device}")
        with self._reserved(sequences, [n] * B) as (slots, positions, _, table, lengths):
            # a draft's position: the context, and the drafts it follows
            positions = (positions.view(B, n)[:, :1] + tree.sum(1) - 1).flatten()

            def attend(q, keys, values):
                return decoder.cache_attention(q.view(B, n, -1, self.head_dim), keys, values, table, lengths, tree=tree)

            return self._layers(x.reshape(B * n, H), positions, slots, attend).view(B, n, H)

    def keep(self, sequences, paths, drafts: int):
        """paths[i]: the numbers of the drafts of sequences[i], of ``drafts``, that are
        accepted, increasing."""
        from .pages import keep_drafts

        paths = [[int(d) for d in path] for path in paths]
        if len(set(sequences)) < len(sequences):
            raise ValueError("keep takes a sequence once")
        if any(self.pool.length(s) < drafts for s in sequences):
            raise ValueError(f"a sequence has fewer than {drafts} tokens")
        if not all(self.pool.alone(s, drafts) for s in sequences):
            raise ValueError("a fork holds the drafts' pages: keep comes before it")
        if len(paths) != len(sequences) or any(sorted(set(p)) != p or any(not 0 <= d < drafts for d in p) for p in paths):
            raise ValueError(f"paths must hold increasing numbers of drafts below {drafts}, one path a sequence")
        table, lengths = self.pool.table(sequences)
        width = max([1, *map(len, paths)])
        path = self.pool._tensor([p + [-1] * (width - len(p)) for p in paths], lengths.dtype)
        keep_drafts(self.pool.caches, table, lengths, path.view(len(paths), width), drafts)
        for s, p in zip(sequences, paths):
            self.pool.trim(s, self.pool.length(s) - drafts + len(p))


def _stats(samples) -> dict:
    """The latency keys of bench/e2e_block.py:281-302."""
    samples = sorted(samples)
    return dict(latency_ms_avg=statistics.fmean(samples), latency_ms_p50=statistics.median(samples),
                latency_ms_p90=samples[math.ceil(0.90 * len(samples)) - 1], latency_ms_min=samples[0],
                latency_ms_max=samples[-1], iterations=len(samples))


def _time_model(torch, fn, x, warmup: int, repeats: int) -> dict:
    for _ in range(warmup):
        fn(x)
    torch.cuda.synchronize()
    samples = []
    stream = torch.cuda.current_stream()
    for _ in range(repeats):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record(stream)
        fn(x)
        b.record(stream)
        b.synchronize()
        samples.append(a.elapsed_time(b))
    return _stats(samples)


def bench_model(S: int, cfg: dict, args) -> dict:
    """One sequence length (bench/e2e_block.py:305-356)."""
    import torch

    from . import compat, ops

    compat._positive("S", S)
    if getattr(args, "serve_arm", False):
        compat._positive("serve-sequences", args.serve_sequences)
        compat._positive("serve-chunk", args.serve_chunk)
    H, I, n_heads, kv_heads = cfg["hidden"], cfg["intermediate"], cfg["heads"], cfg["kv_heads"]
    n_layers = args.layers if args.layers is not None else cfg["layers"]
    dev = torch.device("cuda:0")
    dtype = torch.bfloat16
    if args.model_path:
        print(f"S={S}: loading real checkpoint weights for {n_layers} layers...", flush=True)
        weights = load_checkpoint_weights(args.model_path, list(range(n_layers)), dev, dtype)
        R = weights[0]["ug"].shape[1]
        compress_ratio = R / ops.low_rank_dim(H, I, 1.0)
    else:
        R = ops.low_rank_dim(H, I, args.compress_ratio)
        compress_ratio = args.compress_ratio
        gen = torch.Generator(device=dev)
        gen.manual_seed(args.seed)
        weights = [make_layer_weights(gen, dev, H, I, R, n_heads, kv_heads, dtype) for _ in range(n_layers)]
        if cfg.get("head_norms"):
            for w in weights:
                w.update(q_norm_w=torch.ones(H // n_heads, device=dev, dtype=dtype), k_norm_w=torch.ones(H // n_heads, device=dev, dtype=dtype))
    xgen = torch.Generator(device=dev)
    xgen.manual_seed(args.seed ^ 0xDEAD)
    x = (torch.randn((S, H), generator=xgen, device=dev, dtype=torch.float32) * 0.02).to(dtype)
    r_max = max(max(w["ug"].shape[1], w["ud"].shape[1]) for w in weights)  # checkpoint ranks may differ per layer
    workspace = ops.svd_mlp_workspace(x, r=r_max, ff=I)

    def unfused_model(x):
        for w in weights:
            x = unfused_block(x, w, n_heads, kv_heads)
        return x

    def fused_model(x):
        for w in weights:
            x = fused_block(x, w, n_heads, kv_heads, workspace)
        return x

    # both arms first agree on the output (same weights, same rounding points
    # up to accumulation order)
    got, want = fused_model(x).float(), unfused_model(x).float()
    agreement = float(torch.linalg.norm(got - want) / torch.clamp(torch.linalg.norm(want), min=1e-12))
    if not bool(torch.isfinite(got).all()):
        raise FloatingPointError("fused model output contains NaN/Inf")
    unfused_stats = _time_model(torch, unfused_model, x, args.warmup, args.repeats)
    fused_stats = _time_model(torch, fused_model, x, args.warmup, args.repeats)
    rec = dict(seq_len=S, hidden=H, intermediate=I, rank=R, compress_ratio=compress_ratio, num_layers=n_layers,
               num_heads=n_heads, num_kv_heads=kv_heads, weights="checkpoint" if args.model_path else "synthetic",
               unfused_block=unfused_stats, fused_block=fused_stats,
               speedup_fused_vs_unfused=unfused_stats["latency_ms_avg"] / fused_stats["latency_ms_avg"],
               fused_vs_unfused_relative_l2=agreement)
    if args.dense_arm:
        dense = [tuple((w[u].float() @ w[v].float()).to(dtype).t().contiguous()
                       for u, v in (("uu", "vu"), ("ug", "vg"), ("ud", "vd"))) for w in weights]

        def dense_model(x):
            for w, dw in zip(weights, dense):
                x = dense_block(x, w, dw, n_heads, kv_heads)
            return x

        rec["dense_block"] = _time_model(torch, dense_model, x, args.warmup, args.repeats)
        rec["speedup_fused_vs_dense"] = rec["dense_block"]["latency_ms_avg"] / fused_stats["latency_ms_avg"]
        del dense
    if getattr(args, "decoder_arm", False):
        model = DecoderModel(weights, n_heads, kv_heads, S + 1, workspace=workspace)
        want = model.prompt(x)[-1:].float()
        got = model.step(x[-1:], S - 1).float()  # the last token again, by the other attention
        rec["decoder_step_vs_block_relative_l2"] = float(torch.linalg.norm(got - want) / torch.clamp(torch.linalg.norm(want), min=1e-12))
        rec["decoder_block"] = _time_model(torch, model.prompt, x, args.warmup, args.repeats)
        rec["decoder_step"] = _time_model(torch, lambda x: model.step(x, S), x[:1].contiguous(), args.warmup, args.repeats)
    if getattr(args, "serve_arm", False):
        rec["served_step"] = _serve(torch, weights, n_heads, kv_heads, x, args, workspace)
    del weights
    return rec


def _serve(torch, weights, n_heads: int, kv_heads: int, x, args, workspace) -> dict:
    """A server's step: args.serve_sequences sequences of S tokens generate one each, and
    one reads the chunk of args.serve_chunk behind its S tokens.  All have the same
    tokens, each in pages of its own."""
    from . import ops
    from .pages import copy_pages

    S, n, chunk = x.shape[0], args.serve_sequences, args.serve_chunk
    model = SequenceModel(weights, n_heads, kv_heads, n * -(-(S + 1) // SequenceModel.PAGE) + -(-(S + chunk) // SequenceModel.PAGE),
                          workspace=workspace)
    first = model.pool.add()
    for at in range(0, S, chunk):
        out = model.step(x[at:at + chunk], [first], [x[at:at + chunk].shape[0]])
    alone = DecoderModel(weights, n_heads, kv_heads, S, workspace=workspace).prompt(x)[-1].float()
    others = [model.pool.add() for _ in range(n)]
    model.pool.reserve(others, [S] * n)
    source, *copies = model.pool.table([first] + others)[0]
    for pages in copies:
        copy_pages(model.pool.caches, source, pages)
    rows = x[torch.arange(n + chunk, device=x.device) % S].contiguous()
    sequences, tokens = others + [first], [1] * n + [chunk]
    model.workspace = ops.svd_mlp_workspace(rows, r=max(max(w["ug"].shape[1], w["ud"].shape[1]) for w in weights), ff=weights[0]["vg"].shape[1])

    def step(rows):
        model.step(rows, sequences, tokens)
        for s in sequences:
            model.pool.trim(s, S)

    stats = _time_model(torch, step, rows, args.warmup, args.repeats)
    return dict(stats, sequences=n, chunk=chunk,
                chunks_vs_prompt_relative_l2=float(torch.linalg.norm(out[-1].float() - alone) / torch.clamp(torch.linalg.norm(alone), min=1e-12)))


def _parser() -> argparse.ArgumentParser:
    """The flags of bench/e2e_block.py:363-394, plus --dense-arm."""
    p = argparse.ArgumentParser(description="Whole-model N-layer transformer E2E: fused vs unfused SVD MLP.")
    p.add_argument("--model", choices=list(_SHAPES), default="llama3-3b")
    p.add_argument("--seq-lens", type=int, nargs="+", default=[128, 512, 1024], metavar="S")
    p.add_argument("--layers", type=int, default=None, help="Override layer count (default: model depth)")
    p.add_argument("--model-path", type=str, default=None, metavar="PATH",
                   help="Path to an SVD-decomposed HF checkpoint directory. If omitted, synthetic random weights are used.")
    p.add_argument("--compress-ratio", type=float, default=_DEFAULT_COMPRESS_RATIO)
    p.add_argument("--warmup", type=int, default=3)
    p.add_argument("--repeats", type=int, default=10)
    p.add_argument("--seed", type=int, default=42)
    p.add_argument("--output", type=str, default=None, help="Write full JSON report to this path")
    p.add_argument("--dense-arm", action="store_true", help="also time the dense SwiGLU block (weights rebuilt as U.V)")
    p.add_argument("--decoder-arm", action="store_true",
                   help="also time the causal decoder with rotary positions and a paged cache: a prompt, and one more token")
    p.add_argument("--serve-arm", action="store_true",
                   help="also time a step of several sequences side by side: each generates a token, one reads a chunk of its prompt")
    p.add_argument("--serve-sequences", type=int, default=32, metavar="N", help="sequences that generate in the step")
    p.add_argument("--serve-chunk", type=int, default=256, metavar="T", help="tokens of a prompt's chunk")
    return p


def main(argv=None) -> int:
    args = _parser().parse_args(argv)
    import torch

    if not torch.cuda.is_available():
        raise RuntimeError("E2E block benchmark requires a ROCm GPU")
    cfg = _SHAPES[args.model]
    results = []
    for S in args.seq_lens:
        rec = bench_model(S, cfg, args)
        results.append(rec)
        print(json.dumps(rec, indent=2), flush=True)
    report = dict(model=args.model, backend="rocm", torch_version=torch.__version__,
                  devices=[torch.cuda.get_device_name(0)], compress_ratio=args.compress_ratio, cases=results)
    if args.output:
        with open(args.output, "w", encoding="utf-8") as fh:
            json.dump(report, fh, indent=2)
            fh.write("\n")
    return 0


if __name__ == "__main__":
    sys.exit(main())

"""Measured cases of the operators around the MLP block of a decoder layer:
rotary positions, attention over prompts, attention over a paged cache, and
the norms before and after a block with the residual sum.

Every case is one call.  ``own`` false: the operator in its plain form
(elementary torch operations in 32 bits, rounded once at the end); true: the
package's kernels (``svdmlp.rope``, ``rope_append``, ``prompt_attention``,
``cache_attention``, ``residual_norm``).  A case is a dict of

    op         rope     q, k rotated by the tokens' positions; with `page` > 0
                        k (rotated) and v go to the rows of a paged cache
               prompt   attention of packed sequences onto themselves
               cache    attention of `drafts` new tokens a sequence onto the
                        paged cache that holds the context and them
               norm     r = x + scale * gate * post_norm(branch), and norm(r)
    dtype      bf16 or fp32
    heads, kv_heads, head_dim   (rope, prompt, cache)
    tokens     rows (rope, norm), all sequences' tokens together (prompt)
    sequences  how many they are (rope, prompt, cache); lengths by `_lengths`
    rot, interleaved, stretch   rotated part of the head, pair layout, and the
               factor by which positions are stretched for long contexts
    causal     (prompt)
    context    longest sequence in the cache, new tokens among it (cache)
    tree       each sequence's drafts are a tree of its own (cache)
    page       tokens a page of the cache
    d, post, gate, scale        row length, whether the branch is normalised
               first, its gate ("none", "vector", "rows") and its scale (norm)
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = Path(__file__).resolve().parent.parent / "neuronmlp-on-tpu_amd"
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-5
_THETA = 500000.0


def _package():
    if str(_PACKAGE) not in sys.path:
        sys.path.insert(0, str(_PACKAGE))
    import svdmlp

    return svdmlp


def _rope(tokens, heads, kv_heads, head_dim, *, rot=None, interleaved=False, stretch=1.0, page=0, sequences=1, dtype="bf16"):
    return {"op": "rope", "dtype": dtype, "tokens": tokens, "sequences": sequences, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "rot": rot or head_dim, "interleaved": interleaved,
            "stretch": stretch, "page": page}


def _prompt(tokens, sequences, heads, kv_heads, head_dim, *, causal=True, dtype="bf16"):
    return {"op": "prompt", "dtype": dtype, "tokens": tokens, "sequences": sequences, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "causal": causal}


def _cache(sequences, drafts, context, heads, kv_heads, head_dim, *, page, tree=False, dtype="bf16"):
    return {"op": "cache", "dtype": dtype, "sequences": sequences, "drafts": drafts, "context": context,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "tree": tree}


def _norm(tokens, d, *, post=False, gate="none", scale=1.0, dtype="bf16"):
    return {"op": "norm", "dtype": dtype, "tokens": tokens, "d": d, "post": post, "gate": gate, "scale": scale}


def listed():
    return [
        # one new token of each of 16 sequences on its way into the cache: every decode step, every layer
        {"name": "rope-append-16", **_rope(16, 32, 8, 128, page=16, sequences=16)},
        # the packed prompts of a prefill step, positions stretched for a long context
        {"name": "rope-prompt-6007", **_rope(6007, 32, 8, 128, stretch=4.0, sequences=5)},
        # half of the head rotated, neighbouring pairs, in 32 bits (numerics work)
        {"name": "rope-partial-fp32-2501", **_rope(2501, 16, 16, 64, rot=32, interleaved=True, dtype="fp32")},
        # the end-to-end benchmark's own attention: one short 3B prompt, every token seeing every other
        {"name": "prompt-3b-512", **_prompt(512, 1, 24, 8, 128, causal=False)},
        # a prefill step of a server: prompts of very different lengths packed together
        {"name": "prompt-8b-packed-8191", **_prompt(8191, 17, 32, 8, 128)},
        # one long document on an 8B model, the largest call
        {"name": "prompt-8b-16384", **_prompt(16384, 1, 32, 8, 128)},
        # small heads in 32 bits (numerics work, tests)
        {"name": "prompt-fp32-1001", **_prompt(1001, 3, 16, 16, 64, dtype="fp32")},
        # one user's generated token on an 8B model: the latency of every step
        {"name": "cache-8b-decode-1", **_cache(1, 1, 4097, 32, 8, 128, page=16)},
        # a server's ordinary decode step: 64 sequences of different ages
        {"name": "cache-8b-decode-64", **_cache(64, 1, 4096, 32, 8, 128, page=16)},
        # trees of 16 drafted tokens over long contexts on a 70B model
        {"name": "cache-70b-tree-8", **_cache(8, 16, 16384, 64, 8, 128, page=64, tree=True)},
        # residual sum and the next norm of a small decode batch
        {"name": "norm-8b-decode-8", **_norm(8, 4096)},
        # a 70B prompt with a norm on both sides of the block, gated and scaled
        {"name": "norm-70b-prompt-4096", **_norm(4096, 8192, post=True, gate="vector", scale=0.25)},
    ]


_HEADS = ((32, 8, 128), (64, 8, 128), (24, 8, 128), (16, 16, 64), (14, 2, 64), (12, 4, 96), (8, 1, 256), (7, 7, 80))


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    """One more case of the same ranges, of at most the largest listed one's work."""
    op = rng.choice(("rope", "prompt", "cache", "norm"))
    dtype = rng.choice(("bf16",) * 3 + ("fp32",))
    heads, kv_heads, head_dim = rng.choice(_HEADS)
    if op == "rope":
        page = rng.choice((0, 0, 16, 64))
        tokens = _log(rng, 1, 512 if page else 16384)
        rot = rng.choice((head_dim, head_dim, head_dim // 2, head_dim // 4))
        return _rope(tokens, heads, kv_heads, head_dim, rot=rot, interleaved=rng.random() < 0.5,
                     stretch=rng.choice((1.0, 4.0, 8.0)), page=page, sequences=min(tokens, _log(rng, 1, 64)), dtype=dtype)
    if op == "prompt":
        tokens = _log(rng, 1, 12000 if dtype == "bf16" else 4000)
        most = 32 * 16384 * 128 * 16384 // 2
        tokens = min(tokens, int(math.sqrt(most / (heads * head_dim))))
        return _prompt(tokens, min(tokens, _log(rng, 1, 40)), heads, kv_heads, head_dim,
                       causal=rng.random() < 0.75, dtype=dtype)
    if op == "cache":
        sequences = _log(rng, 1, 96)
        context = _log(rng, 1, min(32768, (1 << 18) * 8 // kv_heads // sequences))
        drafts = min(context, rng.choice((1, 1, 1, rng.randint(2, 64))))
        return _cache(sequences, drafts, context, heads, kv_heads, head_dim, page=rng.choice((16, 16, 32, 64, 48)),
                      tree=drafts > 1 and rng.random() < 0.7, dtype=dtype)
    return _norm(_log(rng, 1, 8192), rng.choice((1024, 2560, 4096, 8192, 3584, 1000)), post=rng.random() < 0.5,
                 gate=rng.choice(("none", "vector", "rows")), scale=rng.choice((1.0, 0.22, 1.4)), dtype=dtype)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(total, parts):
    """`parts` lengths of different size, at least 1, that sum to `total`."""
    rng = random.Random(total * 8191 + parts)
    weights = [rng.uniform(0.05, 1.0) for _ in range(parts)]
    lens = [max(1, int(total * w / sum(weights))) for w in weights]
    while sum(lens) != total:  # what the rounding left goes to, or comes from, the longest
        i = max(range(parts), key=lambda j: lens[j])
        lens[i] = max(1, lens[i] + total - sum(lens))
    return lens


def _contexts(case):
    """Cached tokens a sequence: the first is the longest, the others from a sixteenth of it on."""
    rng = random.Random(case["context"] * 131 + case["sequences"])
    most, n = case["context"], case["drafts"]
    return [most] + [max(n, rng.randint(max(1, most // 16), most)) for _ in range(case["sequences"] - 1)]


def _inv_freq(case, device):
    half = case["rot"] // 2
    return _THETA ** (-torch.arange(half, dtype=torch.float64, device=device) / half) / case["stretch"]


def _attention_factor(case):
    """The factor on cos and sin that goes with stretched positions."""
    return 1.0 if case["stretch"] == 1.0 else 1.0 + 0.1 * math.log(case["stretch"])


def _pages(g, counts, spare):
    """A block table (sequences, most pages of one) of shuffled pages, and how many pages there are."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g, device=g.device).to(torch.int32)
    table = torch.zeros((len(counts), max(counts)), dtype=torch.int32, device=g.device)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    return table, total


def _tree(rng, n):
    """Which drafts each of n drafts sees: itself and its ancestors, parents drawn among the earlier ones."""
    mask = [[False] * n for _ in range(n)]
    for i in range(n):
        if i:
            mask[i] = list(mask[rng.randrange(max(0, i - 6), i)])
        mask[i][i] = True
    return mask


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=g.device, dtype=torch.float32).to(dtype)

    state = {"case": case}
    if case["op"] == "norm":
        T, d = case["tokens"], case["d"]
        spread = torch.exp(0.5 * torch.randn(d, generator=g, device=g.device))
        state["x"] = (torch.randn(T, d, generator=g, device=g.device) * spread).to(dtype)
        state["branch"] = randn(T, d)
        state["weight"] = torch.rand(d, generator=g, device=g.device) * 0.2 + 0.9
        state["post"] = torch.rand(d, generator=g, device=g.device) * 0.2 + 0.9 if case["post"] else None
        state["gate"] = {"none": None, "vector": randn(d), "rows": randn(T, d)}[case["gate"]]
        return state
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] in ("rope", "prompt"):
        T = case["tokens"]
        lens = _lengths(T, case["sequences"])
        qkv = randn(T, (H + 2 * K) * D)  # what the fused projection wrote
        state["q"] = qkv[:, :H * D].view(T, H, D)
        state["k"] = qkv[:, H * D:(H + K) * D].view(T, K, D)
        state["v"] = qkv[:, (H + K) * D:].view(T, K, D)
        ends = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        state["cu"] = ends.to(g.device)
        state["longest"] = max(lens)
        if case["op"] == "rope":
            state["inv_freq"] = _inv_freq(case, g.device)
            state["scale"] = _attention_factor(case)
            start = torch.randint(0, 8192, (len(lens),), generator=g, device=g.device)
            within = torch.cat([torch.arange(n) for n in lens]).to(g.device)
            seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(g.device)
            state["positions"] = start[seq] + within
            if case["page"]:
                pages = 4 * -(-T // case["page"]) + 256
                state["k_cache"] = randn(pages, case["page"], K, D)
                state["v_cache"] = randn(pages, case["page"], K, D)
                state["slots"] = torch.randperm(pages * case["page"], generator=g, device=g.device)[:T]
        return state
    B, n, page = case["sequences"], case["drafts"], case["page"]
    lens = _contexts(case)
    state["q"] = randn(B, n, H, D)
    state["table"], pages = _pages(g, [-(-c // page) for c in lens], 16)
    state["k_cache"], state["v_cache"] = randn(pages, page, K, D), randn(pages, page, K, D)
    state["lengths"] = torch.tensor(lens, dtype=torch.int32).to(g.device)
    state["tree"] = None
    if case["tree"]:
        rng = random.Random(seed)
        state["tree"] = torch.tensor([_tree(rng, n) for _ in range(B)]).to(g.device)
    return state


# ---------------------------------------------------------------------------
# The operators: the package's calls, and their plain forms
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _own_rope, "prompt": _own_prompt, "cache": _own_cache, "norm": _own_norm}[op](state)
    return {"rope": _plain_rope, "prompt": _plain_prompt, "cache": _plain_cache, "norm": _plain_norm}[op](state)


def _own_rope(s):
    svdmlp, case = _package(), s["case"]
    if case["page"]:
        q = svdmlp.rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"], s["slots"],
                               interleaved=case["interleaved"], scale=s["scale"])
        return q, s["k_cache"], s["v_cache"]
    return svdmlp.rope(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=case["interleaved"], scale=s["scale"])


def _own_prompt(s):
    return _package().prompt_attention(s["q"], s["k"], s["v"], s["cu"], causal=s["case"]["causal"])


def _own_cache(s):
    return _package().cache_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], tree=s["tree"])


def _own_norm(s):
    return _package().residual_norm(s["x"], s["branch"], s["weight"], post_weight=s["post"], gate=s["gate"],
                                    scale=s["case"]["scale"], eps=_EPS)


def _rotate(x, cos, sin, rot, interleaved):
    x32 = x.float()
    part = x32[..., :rot]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x32[..., rot:]), dim=-1).to(x.dtype)


def _plain_rope(s):
    case = s["case"]
    angles = s["positions"].double()[:, None] * s["inv_freq"]  # far positions: 64 bits
    cos = (angles.cos() * s["scale"]).float()[:, None, :]
    sin = (angles.sin() * s["scale"]).float()[:, None, :]
    q = _rotate(s["q"], cos, sin, case["rot"], case["interleaved"])
    k = _rotate(s["k"], cos, sin, case["rot"], case["interleaved"])
    if not case["page"]:
        return q, k
    s["k_cache"].flatten(0, 1)[s["slots"]] = k
    s["v_cache"].flatten(0, 1)[s["slots"]] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _attend(q, k, v, hidden):
    """Softmax attention in 32 bits: q (B, L, H, D) on k, v (B, S, K, D); hidden (B, 1, L or 1, S): keys not seen."""
    B, L, H, D = q.shape
    S, K = k.shape[1], k.shape[2]
    group = H // K
    q = q.float().view(B, L, K, group, D).permute(0, 2, 3, 1, 4).reshape(B, K, group * L, D)
    scores = torch.matmul(q, k.float().permute(0, 2, 3, 1).contiguous())
    scores.mul_(1.0 / math.sqrt(D))
    scores = scores.view(B, H, L, S).masked_fill_(hidden, -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    scores.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores.view(B, K, group * L, S), v.float().permute(0, 2, 1, 3).contiguous())
    out = out.view(B, H, L, D) / torch.where(total == 0, 1.0, total)
    return out.transpose(1, 2)


def _plain_prompt(s):
    q, cu, longest = s["q"], s["cu"].long(), s["longest"]
    lens = cu[1:] - cu[:-1]
    at = torch.arange(longest, device=q.device)
    valid = at < lens[:, None]                                  # (B, longest)
    rows = torch.where(valid, cu[:-1, None] + at, 0)
    hidden = ~valid[:, None, None, :]
    if s["case"]["causal"]:
        hidden = hidden | (at[None, :] > at[:, None])
    out = _attend(q[rows], s["k"][rows], s["v"][rows], hidden)  # (B, longest, H, D)
    token = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu[1:], token, right=True)
    return out[seq, token - cu[seq]].to(q.dtype)


def _plain_cache(s):
    q, table, lens = s["q"], s["table"].long(), s["lengths"].long()
    B, n = q.shape[:2]
    page = s["case"]["page"]
    at = torch.arange(table.shape[1] * page, device=q.device)
    draft = at - (lens[:, None] - n)                            # (B, S): which draft a key is, negative: the context
    if s["tree"] is None:
        seen = draft[:, None, :] <= torch.arange(n, device=q.device)[:, None]
    else:
        index = draft.clamp(0, n - 1)[:, None, :].expand(B, n, -1)
        seen = (draft < 0)[:, None, :] | (torch.gather(s["tree"], 2, index) & (draft < n)[:, None, :])
    k, v = s["k_cache"][table].flatten(1, 2), s["v_cache"][table].flatten(1, 2)
    return _attend(q, k, v, ~seen[:, None]).to(q.dtype)


def _plain_norm(s):
    x, branch = s["x"].float(), s["branch"].float()
    if s["post"] is not None:
        branch = branch * torch.rsqrt((branch * branch).mean(dim=-1, keepdim=True) + _EPS) * s["post"]
    if s["gate"] is not None:
        branch = branch * s["gate"].float()
    r = x + s["case"]["scale"] * branch
    n = r * torch.rsqrt((r * r).mean(dim=-1, keepdim=True) + _EPS) * s["weight"]
    return r.to(s["x"].dtype), n.to(s["x"].dtype)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        T, d = case["tokens"], case["d"]
        rows = 4 + (case["gate"] == "rows")
        vectors = 4 * d * (1 + case["post"]) + (e * d if case["gate"] == "vector" else 0)
        return {"bytes": rows * T * d * e + vectors, "flops": T * d * (8 + 4 * case["post"])}
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        T = case["tokens"]
        moved = 2 * T * (H + K) * D * e + 8 * T + 4 * case["rot"]
        if case["page"]:
            moved += 2 * T * K * D * e + 8 * T
        return {"bytes": moved, "flops": T * (H + K) * case["rot"] * 3}
    if case["op"] == "prompt":
        lens = _lengths(case["tokens"], case["sequences"])
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        return {"bytes": (2 * H + 2 * K) * case["tokens"] * D * e, "flops": 4 * D * H * pairs}
    lens, n = _contexts(case), case["drafts"]
    return {"bytes": 2 * sum(lens) * K * D * e + 2 * case["sequences"] * n * H * D * e,
            "flops": 4 * D * H * n * sum(lens)}


# ---------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_rope(s):
    case = s["case"]
    R, H = case["rot"], case["rot"] // 2
    pairs = [(2 * p, 2 * p + 1) if case["interleaved"] else (p, p + H) for p in range(H)]
    first, second = [a for a, _ in pairs], [b for _, b in pairs]
    theta = torch.outer(s["positions"].double(), s["inv_freq"].double())
    turn = torch.polar(torch.full_like(theta, s["scale"]), theta)  # each pair as a complex number, turned

    def turned(x):
        y = x.double().clone()
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None, :]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = turned(s["q"]), turned(s["k"])
    if not case["page"]:
        return q, k
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    page, slot = s["slots"] // case["page"], s["slots"] % case["page"]
    kc[page, slot], vc[page, slot] = k, s["v"].double()
    return q, kc, vc


def _exact_rows(q, k, v, seen):
    """softmax(q k^T / sqrt(D)) v of one head in 64 bits, in stripes of rows; seen(first, last): the rows' visible keys, or None."""
    D = q.shape[-1]
    out = torch.zeros_like(q)
    for a in range(0, q.shape[0], 4096):
        b = min(q.shape[0], a + 4096)
        w = q[a:b] @ k.t().contiguous() / math.sqrt(D)
        mask = seen(a, b)
        if mask is not None:
            w[~mask] = -math.inf
        out[a:b] = torch.softmax(w, dim=-1) @ v
    return out


def _exact_prompt(s):
    case = s["case"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    at = 0
    for n in _lengths(case["tokens"], case["sequences"]):
        keys = torch.arange(n, device=q.device)
        for h in range(case["heads"]):
            rows = slice(at, at + n)
            out[rows, h] = _exact_rows(q[rows, h].contiguous(), k[rows, h // group].contiguous(), v[rows, h // group].contiguous(),
                                       lambda a, b: keys[None, :] <= keys[a:b, None] if case["causal"] else None)
        at += n
    return out


def _exact_cache(s):
    case = s["case"]
    n, group, page = case["drafts"], case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, length in enumerate(_contexts(case)):
        held = s["table"][b, :-(-length // page)].long()
        k = s["k_cache"][held].flatten(0, 1)[:length].double()
        v = s["v_cache"][held].flatten(0, 1)[:length].double()
        seen = torch.ones((n, length), dtype=torch.bool, device=k.device)
        among = torch.ones((n, n), dtype=torch.bool, device=k.device).tril() if s["tree"] is None else s["tree"][b]
        seen[:, length - n:] = among
        for h in range(case["kv_heads"]):
            q = s["q"][b, :, h * group:(h + 1) * group].double().reshape(n * group, -1)
            rows = seen.repeat_interleave(group, dim=0)
            out[b, :, h * group:(h + 1) * group] = _exact_rows(q, k[:, h].contiguous(), v[:, h].contiguous(),
                                                               lambda a, z: rows[a:z]).view(n, group, -1)
    return out


def _exact_norm(s):
    def rms(t):
        return torch.linalg.vector_norm(t, dim=1, keepdim=True).square() / t.shape[1]

    b = s["branch"].double()
    if s["post"] is not None:
        b = b / (rms(b) + _EPS).sqrt() * s["post"].double()
    if s["gate"] is not None:
        b = b * s["gate"].double()
    r = s["x"].double() + b * s["case"]["scale"]
    return r, r / (rms(r) + _EPS).sqrt() * s["weight"].double()


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "prompt": _exact_prompt, "cache": _exact_cache, "norm": _exact_norm}[case["op"]](s)

"""Measured cases of what serves chunks of prompts, drafts and forks from a
paged cache: norms of the heads with the rotary positions in one pass, attention
of packed chunks of new tokens over the cache, copies of its pages, and the rows
of accepted drafts moved behind the context.

Every case is one call.  ``own`` false: the operator in its plain form
(elementary torch operations in 32 bits, rounded once at the end); true: the
package's kernels (``svdmlp.norm_rope``, ``norm_rope_append``,
``chunk_attention``, ``copy_pages``, ``keep_drafts``).  A case is a dict of

    op         norms    q, k normalised a head and rotated by the tokens' positions;
                        with `page` > 0 k and v go to the rows of a paged cache
               chunk    attention of each sequence's new tokens over its part of a
                        paged cache, which holds its context and them
               copy     pages to other pages, in every layer's caches
               keep     accepted drafts' rows to behind the context, in every layer's
    dtype      bf16 or fp32
    kv_heads, head_dim; heads (norms, chunk)
    tokens     rows (norms), new tokens of all sequences together (chunk)
    sequences  how many they are (norms, chunk, keep)
    rot, interleaved   rotated part of the head and pair layout (norms)
    per_head   each head has gains of its own (norms)
    decoding   of the sequences, those with a single new token (chunk)
    context    longest sequence in the cache, new tokens among it (chunk, keep)
    page       tokens a page of the cache
    caches     keys' and values' caches of all layers (copy, keep)
    pages      pages of each (copy)
    moved      pages that are copied (copy)
    partly     of each page only its first rows are held (copy)
    drafts     new tokens a sequence (keep)
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
_EPS = 1e-6
_THETA = 1000000.0


def _package():
    if str(_PACKAGE) not in sys.path:
        sys.path.insert(0, str(_PACKAGE))
    import svdmlp

    return svdmlp


def _norms(tokens, heads, kv_heads, head_dim, *, rot=None, interleaved=False, per_head=False, page=0, sequences=1, dtype="bf16"):
    return {"op": "norms", "dtype": dtype, "tokens": tokens, "sequences": sequences, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rot": rot or head_dim, "interleaved": interleaved, "per_head": per_head, "page": page}


def _chunk(tokens, sequences, decoding, context, heads, kv_heads, head_dim, *, page, dtype="bf16"):
    return {"op": "chunk", "dtype": dtype, "tokens": tokens, "sequences": sequences, "decoding": decoding, "context": context,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page}


def _copy(caches, pages, moved, page, kv_heads, head_dim, *, partly=False, dtype="bf16"):
    return {"op": "copy", "dtype": dtype, "caches": caches, "pages": pages, "moved": moved, "page": page, "kv_heads": kv_heads,
            "head_dim": head_dim, "partly": partly}


def _keep(caches, sequences, drafts, context, page, kv_heads, head_dim, *, dtype="bf16"):
    return {"op": "keep", "dtype": dtype, "caches": caches, "sequences": sequences, "drafts": drafts, "context": context,
            "page": page, "kv_heads": kv_heads, "head_dim": head_dim}


def listed():
    return [
        # one new token of each of 16 sequences on its way into the cache: every decode step, every layer
        {"name": "norms-append-16", **_norms(16, 32, 8, 128, page=16, sequences=16)},
        # the packed chunks of a large prefill step
        {"name": "norms-prompt-6007", **_norms(6007, 32, 8, 128, sequences=5)},
        # half of the head rotated, neighbouring pairs, gains of each head, in 32 bits (numerics work)
        {"name": "norms-partial-fp32-2501", **_norms(2501, 16, 16, 64, rot=32, interleaved=True, per_head=True, dtype="fp32")},
        # the follow-up questions of three users, a few words each: the smallest calls
        {"name": "chunk-8b-37", **_chunk(37, 3, 0, 1000, 32, 8, 128, page=16)},
        # a server's ordinary step: 63 sequences generate, the 64th's prompt comes in chunks
        {"name": "chunk-8b-step-64", **_chunk(512, 64, 63, 4096, 32, 8, 128, page=16)},
        # a chunk of a long document, late in it
        {"name": "chunk-8b-512-of-32768", **_chunk(512, 1, 0, 32768, 32, 8, 128, page=16)},
        # long chunks of four long prompts on a 70B model, the largest call
        {"name": "chunk-70b-8192", **_chunk(8192, 4, 0, 16384, 64, 8, 128, page=64)},
        # small heads in 32 bits, pages of no power of two (numerics work, tests)
        {"name": "chunk-fp32-701", **_chunk(701, 3, 0, 2500, 16, 16, 64, page=48, dtype="fp32")},
        # eight answers branch off one prompt: the partly filled page of each, in the 32 layers of an 8B model
        {"name": "fork-8b-8", **_copy(64, 256, 8, 16, 8, 128, partly=True)},
        # a cache's far pages go to free ones at its front, so that its end can be given back
        {"name": "compact-8b-500", **_copy(64, 1200, 500, 16, 8, 128)},
        # after a step that verified 8 drafts of each of 16 sequences, on an 8B model
        {"name": "keep-8b-16x8", **_keep(64, 16, 8, 300, 16, 8, 128)},
        # trees of 64 drafts of many sequences
        {"name": "keep-8b-128x64", **_keep(32, 128, 64, 220, 16, 8, 128)},
    ]


_HEADS = ((32, 8, 128), (64, 8, 128), (24, 8, 128), (16, 16, 64), (14, 2, 64), (12, 4, 96), (8, 1, 256), (7, 7, 80))


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    """One more case of the same ranges, of at most the largest listed one's work."""
    op = rng.choice(("norms", "chunk", "chunk", "copy", "keep"))
    dtype = rng.choice(("bf16",) * 3 + ("fp32",))
    heads, kv_heads, head_dim = rng.choice(_HEADS)
    page = rng.choice((16, 16, 32, 64, 48, 8))
    if op == "norms":
        into = rng.choice((0, page))
        tokens = _log(rng, 1, 512 if into else 16384)
        return _norms(tokens, heads, kv_heads, head_dim, rot=rng.choice((head_dim, head_dim, head_dim // 2)), interleaved=rng.random() < 0.5,
                      per_head=rng.random() < 0.25, page=into, sequences=min(tokens, _log(rng, 1, 64)), dtype=dtype)
    if op == "chunk":
        sequences = _log(rng, 1, 96)
        decoding = rng.choice((0, sequences // 2, sequences - 1))
        context = _log(rng, 16, min(32768, (1 << 18) * 8 // kv_heads // sequences))
        chunks = sequences - decoding
        most = min(8192, chunks * context) if dtype == "bf16" else min(2048, chunks * context)
        tokens = decoding + max(chunks, _log(rng, chunks, most))
        case = _chunk(tokens, sequences, decoding, context, heads, kv_heads, head_dim, page=page, dtype=dtype)
        while sequences * max(_news(case)) * heads * context > 1 << 33:  # scores that the plain form has room for
            case["tokens"] = decoding + max(chunks, (case["tokens"] - decoding) // 2)
        return case
    if op == "copy":
        caches = rng.choice((8, 28, 56, 64))
        moved = _log(rng, 1, (1 << 30) // (caches * page * kv_heads * head_dim * 4))
        return _copy(caches, 2 * moved + rng.randint(1, 99), moved, page, kv_heads, head_dim, partly=rng.random() < 0.5, dtype=dtype)
    caches = rng.choice((8, 28, 56, 64))
    sequences, drafts = _log(rng, 1, 96), rng.randint(2, 64)
    most = (1 << 30) // (caches * sequences * kv_heads * head_dim * 4)
    return _keep(caches, sequences, drafts, drafts + _log(rng, 1, max(64, min(2000, most))), page, kv_heads, head_dim, dtype=dtype)


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


def _news(case):
    """New tokens a sequence: those that decode come first."""
    return [1] * case["decoding"] + _lengths(case["tokens"] - case["decoding"], case["sequences"] - case["decoding"])


def _held(case, news):
    """Tokens that the cache holds of each sequence, new ones among them: the last has the longest context."""
    rng = random.Random(case["context"] * 131 + case["sequences"])
    most = case["context"]
    return [max(n, rng.randint(max(1, most // 16), most)) for n in news[:-1]] + [max(news[-1], most)]


def _accepted(case, seed):
    """The accepted path of each sequence's tree of drafts: increasing numbers of drafts."""
    rng, n = random.Random(seed * 31 + case["drafts"]), case["drafts"]
    return [sorted(rng.sample(range(n), rng.randint(1, max(1, min(n, 12))))) for _ in range(case["sequences"])]


def _pages(g, counts, spare):
    """A block table (sequences, most pages of one) of shuffled pages, and how many pages there are."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g, device=g.device).to(torch.int32)
    width, starts = max(counts), torch.tensor([0] + counts, device=g.device).cumsum(0)
    at = torch.arange(width, device=g.device)
    there = at < (starts[1:] - starts[:-1])[:, None]
    return torch.where(there, order[torch.where(there, starts[:-1, None] + at, 0)], 0).contiguous(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=g.device, dtype=torch.float32).to(dtype)

    state = {"case": case}
    K, D, page = case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] in ("copy", "keep"):
        if case["op"] == "copy":
            pages, n = case["pages"], case["moved"]
            order = torch.randperm(pages, generator=g, device=g.device).to(torch.int32)
            state["src"], state["dst"] = order[:n].contiguous(), order[n:2 * n].contiguous()
            state["rows"] = torch.randint(1, page, (n,), generator=g, device=g.device, dtype=torch.int32) if case["partly"] else None
        else:
            lens = _held(case, [case["drafts"]] * case["sequences"])
            state["table"], pages = _pages(g, [-(-c // page) for c in lens], 4)
            state["lengths"] = torch.tensor(lens, dtype=torch.int32).to(g.device)
            paths = _accepted(case, seed)
            longest = max(map(len, paths))
            state["path"] = torch.tensor([p + [-1] * (longest - len(p)) for p in paths], dtype=torch.int32).to(g.device)
        state["pool"] = randn(case["caches"], pages, page, K, D)  # the caches of all layers
        return state
    H, T = case["heads"], case["tokens"]
    if case["op"] == "norms":
        lens = _lengths(T, case["sequences"])
        qkv = randn(T, (H + 2 * K) * D) * 3  # what the fused projection wrote
        state["q"] = qkv[:, :H * D].view(T, H, D)
        state["k"] = qkv[:, H * D:(H + K) * D].view(T, K, D)
        state["v"] = qkv[:, (H + K) * D:].view(T, K, D)
        for name, heads in (("q_weight", H), ("k_weight", K)):
            shape = (heads, D) if case["per_head"] else (D,)
            state[name] = torch.rand(shape, generator=g, device=g.device) + 0.5
        state["inv_freq"] = _THETA ** (-torch.arange(case["rot"] // 2, dtype=torch.float64, device=g.device) / (case["rot"] // 2))
        start = torch.randint(0, 8192, (len(lens),), generator=g, device=g.device)
        within = torch.cat([torch.arange(n) for n in lens]).to(g.device)
        seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(g.device)
        state["positions"] = start[seq] + within
        if page:
            pages = 4 * -(-T // page) + 256
            state["k_cache"], state["v_cache"] = randn(pages, page, K, D), randn(pages, page, K, D)
            state["slots"] = torch.randperm(pages * page, generator=g, device=g.device)[:T]
        return state
    news = _news(case)
    lens = _held(case, news)
    state["q"] = randn(T, H, D)
    state["table"], pages = _pages(g, [-(-c // page) for c in lens], 16)
    state["k_cache"], state["v_cache"] = randn(pages, page, K, D), randn(pages, page, K, D)
    state["lengths"] = torch.tensor(lens, dtype=torch.int32).to(g.device)
    state["cu"] = torch.tensor([0] + news, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(g.device)
    state["longest"] = max(news)
    return state


# ---------------------------------------------------------------------------
# The operators: the package's calls, and their plain forms
# ---------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"norms": _own_norms, "chunk": _own_chunk, "copy": _own_copy, "keep": _own_keep}[op](state)
    return {"norms": _plain_norms, "chunk": _plain_chunk, "copy": _plain_copy, "keep": _plain_keep}[op](state)


def _own_norms(s):
    svdmlp, case = _package(), s["case"]
    if case["page"]:
        q = svdmlp.norm_rope_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"], s["k_cache"],
                                    s["v_cache"], s["slots"], eps=_EPS, interleaved=case["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    return svdmlp.norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"], eps=_EPS,
                            interleaved=case["interleaved"])


def _own_chunk(s):
    return _package().chunk_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["cu"])


def _own_copy(s):
    _package().copy_pages(s["pool"], s["src"], s["dst"], s["rows"])
    return s["pool"]


def _own_keep(s):
    return s["pool"], _package().keep_drafts(s["pool"], s["table"], s["lengths"], s["path"], s["case"]["drafts"])


def _normed(x, weight):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + _EPS) * weight


def _rotate(x, cos, sin, rot, interleaved):
    part = x[..., :rot]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., rot:]), dim=-1)


def _plain_norms(s):
    case, dtype = s["case"], s["q"].dtype
    angles = s["positions"].double()[:, None] * s["inv_freq"]  # far positions: 64 bits
    cos, sin = angles.cos().float()[:, None, :], angles.sin().float()[:, None, :]
    q = _rotate(_normed(s["q"], s["q_weight"]), cos, sin, case["rot"], case["interleaved"]).to(dtype)
    k = _rotate(_normed(s["k"], s["k_weight"]), cos, sin, case["rot"], case["interleaved"]).to(dtype)
    if not case["page"]:
        return q, k
    s["k_cache"].flatten(0, 1)[s["slots"]] = k
    s["v_cache"].flatten(0, 1)[s["slots"]] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _attend(q, k, v, hidden):
    """Softmax attention in 32 bits: q (B, L, H, D) on k, v (B, S, K, D); hidden (B, 1, L, S): keys not seen."""
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


def _plain_chunk(s):
    q, cu, table, lens = s["q"], s["cu"].long(), s["table"].long(), s["lengths"].long()
    news = cu[1:] - cu[:-1]
    at = torch.arange(s["longest"], device=q.device)
    rows = torch.where(at < news[:, None], cu[:-1, None] + at, 0)
    place = (lens - news)[:, None] + at                                    # (B, longest): where in its sequence a token is
    keys = torch.arange(table.shape[1] * s["case"]["page"], device=q.device)
    k, v = s["k_cache"][table].flatten(1, 2), s["v_cache"][table].flatten(1, 2)
    out = _attend(q[rows], k, v, (keys > place[:, :, None])[:, None])      # (B, longest, H, D)
    token = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu[1:], token, right=True)
    return out[seq, token - cu[seq]].to(q.dtype)


def _plain_copy(s):
    pool, src, dst = s["pool"], s["src"].long(), s["dst"].long()
    pages = pool[:, src]
    if s["rows"] is not None:
        held = torch.arange(pool.shape[2], device=pool.device) < s["rows"][:, None]
        pages = torch.where(held[None, :, :, None, None], pages, pool[:, dst])
    pool[:, dst] = pages
    return pool


def _plain_keep(s):
    pool, path, page = s["pool"], s["path"].long(), s["case"]["page"]
    context = s["lengths"].long() - s["case"]["drafts"]
    kept = path >= 0
    to = context[:, None] + torch.arange(path.shape[1], device=pool.device)
    to, at = torch.where(kept, to, to[:, :1]), torch.where(kept, context[:, None] + path, (context[:, None] + path)[:, :1])

    def slot(x):  # (behind the last accepted draft: the first one again)
        return torch.gather(s["table"].long(), 1, x // page) * page + x % page

    flat = pool.flatten(1, 2)
    flat[:, slot(to)] = flat[:, slot(at)]
    return pool, (context + kept.sum(dim=1)).to(torch.int32)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    K, D, page = case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "norms":
        T, H = case["tokens"], case["heads"]
        moved = 2 * T * (H + K) * D * e + 8 * T + 4 * case["rot"]
        moved += 4 * D * (H + K if case["per_head"] else 2)
        if page:
            moved += 2 * T * K * D * e + 8 * T
        return {"bytes": moved, "flops": T * (H + K) * (4 * D + 3 * case["rot"])}
    if case["op"] == "chunk":
        news = _news(case)
        lens = _held(case, news)
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(news, lens))
        return {"bytes": 2 * sum(lens) * K * D * e + 2 * case["tokens"] * case["heads"] * D * e, "flops": 4 * D * case["heads"] * pairs}
    if case["op"] == "copy":
        rows = page / 2 if case["partly"] else page
        return {"bytes": 2 * case["caches"] * case["moved"] * rows * K * D * e, "flops": 0}
    rows = sum(map(len, _accepted(case, 0)))
    return {"bytes": 2 * case["caches"] * rows * K * D * e, "flops": 0}


# ---------------------------------------------------------------------------
# The definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_norms(s):
    case = s["case"]
    half = case["rot"] // 2
    pairs = [(2 * p, 2 * p + 1) if case["interleaved"] else (p, p + half) for p in range(half)]
    first, second = [a for a, _ in pairs], [b for _, b in pairs]
    theta = torch.outer(s["positions"].double(), s["inv_freq"].double())
    turn = torch.polar(torch.ones_like(theta), theta)  # each pair as a complex number, turned

    def turned(x, weight):
        x = x.double()
        rms = (torch.linalg.vector_norm(x, dim=-1, keepdim=True).square() / x.shape[-1] + _EPS).sqrt()
        y = x / rms * weight.double()
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None, :]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"])
    if not case["page"]:
        return q, k
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    page, row = s["slots"] // case["page"], s["slots"] % case["page"]
    kc[page, row], vc[page, row] = k, s["v"].double()
    return q, kc, vc


def _exact_chunk(s):
    case, q = s["case"], s["q"]
    group, page, D = case["heads"] // case["kv_heads"], case["page"], case["head_dim"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    news = _news(case)
    first = 0
    for b, (n, m) in enumerate(zip(news, _held(case, news))):
        held = s["table"][b, :-(-m // page)].long()
        k = s["k_cache"][held].flatten(0, 1)[:m].double().transpose(0, 1).contiguous()
        v = s["v_cache"][held].flatten(0, 1)[:m].double().transpose(0, 1).contiguous()
        for a in range(0, n, 2048):  # in stripes of rows
            z = min(n, a + 2048)
            later = torch.arange(m, device=q.device)[None, :] > torch.arange(m - n + a, m - n + z, device=q.device)[:, None]
            for h in range(case["heads"]):
                w = q[first + a:first + z, h].double() @ k[h // group].t().contiguous() / math.sqrt(D)
                w[later] = -math.inf
                out[first + a:first + z, h] = torch.softmax(w, dim=-1) @ v[h // group]
        first += n
    return out


def _exact_copy(s):
    pool = s["pool"].double()
    before = s["pool"]
    rows = [pool.shape[2]] * len(s["src"]) if s["rows"] is None else s["rows"].tolist()
    for i, j, n in zip(s["src"].tolist(), s["dst"].tolist(), rows):
        pool[:, j, :n] = before[:, i, :n].double()
    return pool


def _exact_keep(s):
    pool, before, page = s["pool"].double(), s["pool"], s["case"]["page"]
    table, lens = s["table"].tolist(), s["lengths"].tolist()
    new = []
    for b, path in enumerate(s["path"].tolist()):
        path = [p for p in path if p >= 0]
        context = lens[b] - s["case"]["drafts"]
        for i, p in enumerate(path):
            x, y = context + i, context + p
            pool[:, table[b][x // page], x % page] = before[:, table[b][y // page], y % page].double()
        new.append(context + len(path))
    return pool, torch.tensor(new, dtype=torch.int32)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norms": _exact_norms, "chunk": _exact_chunk, "copy": _exact_copy, "keep": _exact_keep}[case["op"]](s)

"""The operators around the MLP block without a GPU: what the C ABI and the
Python entry points refuse before any HIP call, and the frequencies of rotary
positions."""

import ctypes
import math

import pytest
import torch

import svdmlp
from svdmlp import _lib

P = ctypes.c_void_p(256)
BAD = _lib.SVDMLP_EINVAL


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _strides(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _rope(lib, T=4, Hq=4, Hk=2, D=16, rot=16, scale=1.0, dtype=1, flags=0, q=P):
    return lib.svdmlp_rope(q, P, P, P, P, P, None, T, Hq, Hk, D, rot, scale, dtype, flags, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=0), b"positive"), (dict(Hq=5), b"no multiple"), (dict(rot=18), b"turned values"), (dict(rot=7), b"turned values"),
    (dict(rot=0), b"turned values"), (dict(dtype=2), b"dtype"), (dict(flags=2), b"flags"), (dict(q=None), b"null"),
    (dict(scale=math.inf), b"finite"), (dict(D=2048, rot=2048), b"head size"), (dict(T=1 << 40), b"too many"),
])
def test_rope_refusals(lib, kw, msg):
    assert _rope(lib, **kw) == BAD
    assert msg in lib.svdmlp_last_error()


def test_rope_append_refusals(lib):
    def call(slots=P, v=P, pages=4, page=16, T=4):
        return lib.svdmlp_rope_append(P, P, v, P, P, slots, P, P, P, None, T, pages, page, 4, 2, 16, 16, 1.0, 1, 0, None)

    for kw in (dict(slots=None), dict(v=None), dict(pages=0), dict(page=0), dict(T=-1), dict(page=1 << 40), dict(pages=1 << 62)):
        assert call(**kw) == BAD, kw


def _prompt(lib, T=4, B=1, Hq=4, Hk=2, D=16, scale=0.25, dtype=1, flags=1, cu=None, out=P, strides=None):
    return lib.svdmlp_prompt_attention(P, P, P, cu, out, strides, T, B, Hq, Hk, D, scale, dtype, flags, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(T=0), b"positive"), (dict(Hk=3), b"no multiple"), (dict(D=264), b"head size"), (dict(D=12), b"16-byte"),
    (dict(B=2), b"bounds"), (dict(B=0), b"bounds"), (dict(scale=0.0), b"scale"), (dict(scale=math.nan), b"scale"),
    (dict(flags=4), b"flags"), (dict(out=ctypes.c_void_p(264)), b"16-byte"), (dict(out=None), b"null"),
    (dict(strides=_strides(64, 16, 32, 16, 32, 16, 64, 12)), b"16-byte"), (dict(strides=_strides(64, 16, -32, 16, 32, 16, 64, 16)), b"negative"),
    (dict(strides=_strides(64, 16, 32, 16, 1 << 24, 16, 64, 16)), b"apart"), (dict(T=1 << 31), b"too many"), (dict(dtype=2), b"dtype"),
])
def test_prompt_attention_refusals(lib, kw, msg):
    assert _prompt(lib, **kw) == BAD
    assert msg in lib.svdmlp_last_error()


def _cache(lib, B=2, n=1, pages=4, page=16, width=2, Hq=4, Hk=2, D=16, scale=0.25, dtype=1, table=P, ws=None, nbytes=0, counters=None, n_counters=0):
    return lib.svdmlp_cache_attention(P, P, P, table, P, None, P, None, B, n, pages, page, width, Hq, Hk, D, scale, dtype, ws, nbytes, counters, n_counters, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(B=0), b"positive"), (dict(n=0), b"positive"), (dict(n=65), b"at most 64"), (dict(width=0), b"positive"),
    (dict(page=1 << 20, width=1 << 20), b"2^31"), (dict(pages=0), b"positive"), (dict(page=1, width=65537), b"at most 65536"), (dict(D=320), b"head size"),
    (dict(table=None), b"null"), (dict(scale=-1.0), b"scale"), (dict(B=1 << 40), b"too many"),
    (dict(width=4096), b"workspace too small"),  # a long context's partial sums need one
    (dict(width=4096, ws=ctypes.c_void_p(264), nbytes=1 << 30), b"workspace too small"),
    (dict(width=4096, ws=P, nbytes=1 << 30), b"counters needed"), (dict(width=4096, ws=P, nbytes=1 << 30, counters=P, n_counters=3), b"counters needed"),
])
def test_cache_attention_refusals(lib, kw, msg):
    assert _cache(lib, **kw) == BAD
    assert msg in lib.svdmlp_last_error()


def test_cache_attention_workspace(lib):
    counters = ctypes.c_int64(-1)

    def f(*sizes):
        return lib.svdmlp_cache_attention_workspace_bytes(*sizes, 1, ctypes.byref(counters))

    assert f(1, 1, 16, 0, 32, 8, 128) == 0 and counters.value == 0
    assert f(1, 1, 16, 10, 32, 7, 128) == 0 and counters.value == 0
    assert f(1, 1, 16, 1, 32, 8, 128) == 0 and counters.value == 0  # one chunk: no partial sums
    assert f(1, 1, 16, 1 << 13, 32, 8, 128) > 0 and counters.value == 8
    assert f(3, 8, 16, 1 << 13, 64, 8, 128) > 0 and counters.value == 3 * 8  # 64 rows a head: one tile
    assert f(3, 16, 16, 1 << 13, 64, 8, 128) > 0 and counters.value == 0     # over 64 rows: joined by a kernel of its own
    assert lib.svdmlp_cache_attention_workspace_bytes(1, 1, 16, 1 << 13, 32, 8, 128, 1, None) > 0


def test_residual_norm_refusals(lib):
    def call(x=P, b=P, post=None, gate=None, w=P, r=P, n=P, T=4, d=16, scale=1.0, eps=1e-5, dtype=1):
        return lib.svdmlp_residual_norm(x, b, post, gate, w, r, n, None, T, d, scale, eps, dtype, None)

    for kw, msg in ((dict(T=0), b"positive"), (dict(d=32769), b"at most"), (dict(x=None), b"null"), (dict(r=None, n=None), b"null"),
                    (dict(w=None), b"null"), (dict(b=None, gate=P), b"branch"), (dict(b=None, post=P), b"branch"),
                    (dict(eps=0.0), b"eps"), (dict(scale=math.nan), b"scale"), (dict(dtype=2), b"dtype")):
        assert call(**kw) == BAD, kw
        assert msg in lib.svdmlp_last_error(), kw


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def test_python_refusals_before_the_device_is_asked():
    q, k = _t(4, 4, 16), _t(4, 2, 16)
    pos, f = torch.zeros(4, dtype=torch.int64), torch.ones(8, dtype=torch.float64)
    for fn in (lambda: svdmlp.rope(q, k, pos, f), lambda: svdmlp.prompt_attention(q, k, k),
               lambda: svdmlp.residual_norm(_t(2, 8), _t(2, 8), torch.ones(8)),
               lambda: svdmlp.cache_attention(_t(2, 1, 4, 16), _t(4, 16, 2, 16), _t(4, 16, 2, 16),
                                              torch.zeros((2, 1), dtype=torch.int32), torch.ones(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="ROCm GPU"):
            fn()
    with pytest.raises(ValueError, match="no multiple"):
        svdmlp.prompt_attention(_t(4, 5, 16), k, k)
    with pytest.raises(ValueError, match="keys and values"):
        svdmlp.prompt_attention(q, k, _t(3, 2, 16))
    with pytest.raises(TypeError, match="same dtype"):
        svdmlp.prompt_attention(q, k, _t(4, 2, 16, dtype=torch.float32))
    with pytest.raises(TypeError, match="supported dtypes"):
        svdmlp.prompt_attention(*(t.half() for t in (q, k, k)))
    with pytest.raises(ValueError, match="caches must have shape"):
        svdmlp.cache_attention(_t(2, 1, 4, 16), _t(4, 16, 2, 16), _t(5, 16, 2, 16), torch.zeros((2, 1)), torch.ones(2))
    with pytest.raises(ValueError, match="1 to 64"):
        svdmlp.cache_attention(_t(2, 65, 4, 16), _t(4, 16, 2, 16), _t(4, 16, 2, 16), torch.zeros((2, 1)), torch.ones(2))
    with pytest.raises(ValueError, match="without a branch"):
        svdmlp.residual_norm(_t(2, 8), None, None)
    with pytest.raises(ValueError, match="nonempty"):
        svdmlp.residual_norm(_t(0, 8), _t(0, 8), None)


def test_rope_frequencies():
    f, s = svdmlp.rope_frequencies(8, 10000.0)
    assert f.dtype == torch.float64 and s == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    g, s = svdmlp.rope_frequencies(8, 10000.0, scaling={"type": "linear", "factor": 4})
    assert torch.equal(g, f / 4) and s == 1.0
    # ntk: the highest frequency stays, the lowest is divided by the factor
    g, _ = svdmlp.rope_frequencies(64, 10000.0, scaling={"type": "ntk", "factor": 8})
    h, _ = svdmlp.rope_frequencies(64, 10000.0)
    assert g[0] == 1 and math.isclose(float(g[-1] * 8), float(h[-1]), rel_tol=1e-12)
    # by wavelength: short ones kept, long ones stretched, a ramp in between
    g, _ = svdmlp.rope_frequencies(128, 500000.0, scaling=dict(type="llama3", factor=8, low_freq_factor=1,
                                                               high_freq_factor=4, original_context=8192))
    h, _ = svdmlp.rope_frequencies(128, 500000.0)
    wave = 2 * math.pi / h
    assert torch.equal(g[wave < 2048], h[wave < 2048])
    assert torch.allclose(g[wave > 8192], h[wave > 8192] / 8, rtol=1e-14)
    mid = (wave > 2048) & (wave < 8192)
    assert mid.any() and ((g[mid] < h[mid]) & (g[mid] > h[mid] / 8)).all()
    # yarn: the ramp is over the pairs' numbers, and cos and sin grow
    g, s = svdmlp.rope_frequencies(128, 10000.0, scaling=dict(type="yarn", factor=4, original_context=4096))
    h, _ = svdmlp.rope_frequencies(128, 10000.0)
    assert g[0] == h[0] and math.isclose(float(g[-1]), float(h[-1]) / 4, rel_tol=1e-12)
    assert math.isclose(s, 0.1 * math.log(4) + 1)
    assert ((g <= h) & (g >= h / 4 - 1e-18)).all()


@pytest.mark.parametrize("args", [
    dict(rot=7), dict(rot=0), dict(rot=8, theta=1.0), dict(rot=8, scaling={"type": "none of these"}),
    dict(rot=8, scaling={"type": "linear", "factor": 0.5}),
    dict(rot=8, scaling=dict(type="llama3", factor=8, low_freq_factor=4, high_freq_factor=4, original_context=8192)),
])
def test_rope_frequencies_refusals(args):
    with pytest.raises(ValueError):
        svdmlp.rope_frequencies(**args)


def test_e2e_parser_has_the_decoder_arm():
    from svdmlp import e2e_block

    assert e2e_block._parser().parse_args([]).decoder_arm is False
    assert e2e_block._parser().parse_args(["--decoder-arm"]).decoder_arm is True


def test_overlap_of_views():
    """Views of one buffer: told apart exactly where their strides are alike."""
    from svdmlp.decoder import _overlap

    def brute(a, b):
        cells = lambda t: {t.storage_offset() + o for o in (torch.arange(200).as_strided(t.shape, t.stride(), 0)).flatten().tolist()}
        return bool(cells(a) & cells(b))

    x = torch.zeros(200)
    pairs = [(x.view(10, 20)[:, :8], x.view(10, 20)[:, 8:]), (x.view(10, 20)[:, :8], x.view(10, 20)[:, 7:]),
             (x.view(5, 5, 2, 4)[..., 0, :], x.view(5, 5, 2, 4)[..., 1, :]), (x.view(5, 5, 2, 4)[:3, :, 0], x.view(5, 5, 2, 4)[2:, :, 0]),
             (x.view(5, 5, 2, 4)[:2, :, 0], x.view(5, 5, 2, 4)[2:, :, 0]), (x.view(5, 40)[:, :12].view(5, 3, 4), x.view(5, 40)[:, 12:20].view(5, 2, 4)),
             (x.view(5, 40)[:, :12].view(5, 3, 4), x.view(5, 40)[:, 8:16].view(5, 2, 4)), (x[:8].view(1, 2, 4), x[4:12].view(1, 2, 4)),
             (x.view(4, 2, 25)[:, 0], x.view(4, 2, 25)[:, 1]), (x.view(4, 2, 25)[1:, 0], x.view(4, 2, 25)[:3, 1])]
    for a, b in pairs:
        assert _overlap(a, b) == brute(a, b) and _overlap(b, a) == brute(a, b), (a.shape, a.stride(), b.shape, b.storage_offset())

"""What attention over chunks refuses before any HIP call, its workspace, and the options of the layers that call it."""

import ctypes
import math

import pytest
import torch

import svdmlp
from svdmlp import _lib

P = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _strides(**kw):
    s = dict(q=256, qh=64, kp=2048, kt=128, kh=64, vp=2048, vt=128, vh=64, o=256, oh=64, table=4) | kw
    return (ctypes.c_int64 * 11)(*s.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(T=0), b"positive"), (dict(T=1 << 40), b"too"), (dict(Hq=5), b"no multiple"), (dict(Hk=0), b"positive"), (dict(D=264), b"head size"),
    (dict(D=60), b"16-byte"), (dict(dtype=2), b"dtype"), (dict(B=0), b"sequences"), (dict(B=1 << 31), b"sequences"), (dict(pages=0), b"positive"),
    (dict(page=0), b"positive"), (dict(width=-1), b"positive"), (dict(page=1 << 20, width=1 << 20), b"at most"), (dict(width=1 << 31, page=1), b"at most"),
    (dict(scale=0.0), b"scale"), (dict(scale=math.nan), b"scale"), (dict(q=None), b"null"), (dict(cu=None), b"null"), (dict(lengths=None), b"null"),
    (dict(out=ctypes.c_void_p(264)), b"16-byte"), (dict(strides=_strides(kt=-128)), b"negative"), (dict(strides=_strides(vh=60)), b"16-byte"),
    (dict(strides=_strides(kt=1 << 40, kp=1 << 44)), b"apart"), (dict(ws=None, T=4000, width=4000), b"workspace"),
    (dict(nbytes=64, T=4000, width=4000), b"workspace"), (dict(ws=ctypes.c_void_p(264), nbytes=1 << 40, T=4000, width=4000), b"aligned"),
])
def test_chunk_attention_refusals(lib, kw, msg):
    a = dict(q=P, k=P, v=P, table=P, lengths=P, cu=P, out=P, strides=None, T=5, B=2, pages=8, page=16, width=4, Hq=4, Hk=2, D=64, scale=0.1, dtype=1,
             ws=P, nbytes=0) | kw
    assert lib.svdmlp_chunk_attention(*a.values(), None) == _lib.SVDMLP_EINVAL
    assert msg in lib.svdmlp_last_error()


def _bytes(lib, T, B, page, width, Hq, Hk, D, dtype):
    return lib.svdmlp_chunk_attention_workspace_bytes(T, B, page, width, Hq, Hk, D, dtype)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("D", [8, 64, 128, 200, 256])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (32, 8), (64, 8), (7, 7), (128, 1)])
def test_chunk_attention_workspace(lib, dtype, D, Hq, Hk):
    """Never more than two sums of a tile, and a note, for every block that the card holds, whatever the lengths: 256 CUs,
    three blocks each of 32 rows at most, two of 128, one of 256."""
    most = 256 * (3 * (32 + 8 * 32 * (D + 2)) + 2 * (32 + 8 * 128 * (D + 2)) + 32 + 8 * 256 * (D + 2))
    for T in (1, 3, 64, 700, 9000, 1 << 20):
        for B in (1, 2, 64, 65, 1000):
            for page, width in ((1, 1), (16, 300), (64, 4000), (5, 1 << 20)):
                n = _bytes(lib, T, B, page, width, Hq, Hk, D, dtype)
                assert 0 <= n <= most and n % 16 == 0, (T, B, page, width, n)


def test_chunk_attention_workspace_of_bad_sizes(lib):
    for sizes in ((0, 1, 1, 1, 1, 1, 64, 1), (1, 0, 1, 1, 1, 1, 64, 1), (1, 1, 0, 1, 1, 1, 64, 1), (1, 1, 1, 0, 1, 1, 64, 1), (1, 1, 1, 1, 3, 2, 64, 1),
                  (1, 1, 1, 1, 1, 1, 64, 7), (1, 1, 1 << 40, 1 << 40, 1, 1, 64, 1)):
        assert _bytes(lib, *sizes) == 0


def test_chunk_attention_python_refusals_before_the_device_is_asked():
    q, c = torch.zeros(5, 4, 64), torch.zeros(4, 16, 2, 64)
    t, ln, cu = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.tensor([0, 2, 5], dtype=torch.int32)
    for fn, kind, msg in ((lambda: svdmlp.chunk_attention(q, c, c, t, ln, cu), ValueError, "ROCm GPU"),
                          (lambda: svdmlp.chunk_attention(q.half(), c.half(), c.half(), t, ln, cu), TypeError, "dtypes"),
                          (lambda: svdmlp.chunk_attention(q, c.bfloat16(), c.bfloat16(), t, ln, cu), TypeError, "same dtype"),
                          (lambda: svdmlp.chunk_attention(q[0], c, c, t, ln, cu), ValueError, "expected q"),
                          (lambda: svdmlp.chunk_attention(q[:, :3], c, c, t, ln, cu), ValueError, "no multiple")):
        with pytest.raises(kind, match=msg):
            fn()


def test_e2e_parser_has_the_serve_arm():
    from svdmlp import e2e_block

    args = e2e_block._parser().parse_args([])
    assert (args.serve_arm, args.serve_sequences, args.serve_chunk) == (False, 32, 256)
    assert e2e_block._parser().parse_args(["--serve-arm", "--model", "qwen3-8b", "--serve-chunk", "64"]).serve_chunk == 64


@pytest.mark.parametrize("head_norms", [False, True])
def test_checkpoint_weights_with_head_norms(tmp_path, head_norms):
    """The layers' weights from a checkpoint: the gains of the heads too, where it has them."""
    import json

    from safetensors.torch import save_file
    from svdmlp import checkpoint, e2e_block

    D, FF, R, G = 64, 96, 32, torch.Generator().manual_seed(4)
    rand = lambda *shape: torch.randn(shape, generator=G).bfloat16()
    layers = [tuple(rand(*s) for s in ((D, R), (R, FF), (D, R), (R, FF), (FF, R), (R, D))) for _ in range(2)]
    checkpoint.save_mlp_checkpoint(tmp_path, layers, hidden_size=D, intermediate_size=FF)
    more = {}
    for i in range(2):
        p = f"model.layers.{i}."
        more |= {p + "self_attn.q_proj.weight": rand(D, D), p + "self_attn.k_proj.weight": rand(32, D), p + "self_attn.v_proj.weight": rand(32, D),
                 p + "self_attn.o_proj.weight": rand(D, D), p + "input_layernorm.weight": rand(D), p + "post_attention_layernorm.weight": rand(D)}
        if head_norms:
            more |= {p + "self_attn.q_norm.weight": rand(16), p + "self_attn.k_norm.weight": rand(16)}
    save_file(more, str(tmp_path / "attention.safetensors"))
    at = tmp_path / "model.safetensors.index.json"
    index = json.loads(at.read_text())
    index["weight_map"] |= {k: "attention.safetensors" for k in more}
    at.write_text(json.dumps(index))
    for i, w in enumerate(e2e_block.load_checkpoint_weights(tmp_path, [0, 1], "cpu", torch.bfloat16)):
        assert torch.equal(w["wk"], more[f"model.layers.{i}.self_attn.k_proj.weight"].t()) and torch.equal(w["ug"], layers[i][0])
        assert ("q_norm_w" in w) == ("k_norm_w" in w) == head_norms
        if head_norms:
            assert torch.equal(w["q_norm_w"], more[f"model.layers.{i}.self_attn.q_norm.weight"])
            assert torch.equal(w["k_norm_w"], more[f"model.layers.{i}.self_attn.k_norm.weight"])

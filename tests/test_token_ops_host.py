"""Attention, layer norm and embedding lookup, host side (no GPU): the C entry points refuse bad
sizes, types and workspaces before any launch, and the workspace queries answer without touching
memory."""
import ctypes
import os
import struct

import pytest

EINVAL, EWORKSPACE, EDTYPE, ELENGTH, EHEADS = -1, -4, -10, -11, -12


@pytest.fixture(scope="module")
def lib():
    from ttsplat import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from ttsplat import build
        build.build()
    return _lib.load()


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(64)
    return ctypes.cast(buf, ctypes.c_void_p)


def shape(B=1, Hq=2, Hkv=1, Nq=40, Nk=50, D=16, causal=0, dtype=2, ms=0, row=16, scale=0.25):
    st = [Nq * D * Hq, Nq * D, row] * 8
    return struct.pack("=33qd", B, Hq, Hkv, Nq, Nk, D, causal, dtype, ms, *st, scale)


@pytest.mark.parametrize("kw,code", [
    (dict(D=0), EHEADS), (dict(D=129), EHEADS), (dict(Hq=3, Hkv=2), EHEADS),
    (dict(Hkv=0), EINVAL), (dict(B=-1), EINVAL), (dict(Nk=-1), EINVAL),
    (dict(scale=0.0), EINVAL), (dict(scale=float("nan")), EINVAL), (dict(scale=float("inf")), EINVAL),
    (dict(dtype=3), EDTYPE), (dict(dtype=-1), EDTYPE),
    (dict(Nk=1 << 31), ELENGTH), (dict(Nq=1 << 30, Hq=4, Hkv=1), ELENGTH), (dict(row=1 << 23), ELENGTH),
    (dict(B=1 << 20, Hq=1 << 12, Hkv=1 << 12), ELENGTH)])
def test_attention_refuses(lib, p, kw, code):
    s = shape(**kw)
    assert lib.tts_attention_fwd(s, p, p, p, None, p, None, None, None, 0, None) == code
    assert lib.tts_attention_bwd(s, p, p, p, None, p, None, p, p, p, p, p, p, 1 << 40, None) == code
    assert lib.tts_attention_workspace_bytes(s, 0) == 0
    assert lib.tts_strerror(code) != b"unknown error"


def test_attention_pointers_and_workspace(lib, p):
    s = shape()
    assert lib.tts_attention_fwd(None, p, p, p, None, p, None, None, None, 0, None) == EINVAL
    assert lib.tts_attention_fwd(s, p, None, p, None, p, None, None, None, 0, None) == EINVAL
    assert lib.tts_attention_bwd(s, p, p, p, None, p, None, p, p, None, None, None, p, 1 << 40,
                                 None) == EINVAL               # no gradient asked for
    assert lib.tts_attention_bwd(s, p, p, p, None, p, None, p, p, p, p, p, None, 0,
                                 None) == EWORKSPACE
    need = lib.tts_attention_workspace_bytes(s, 1)
    assert need >= 4 * 2 * 40
    assert lib.tts_attention_bwd(s, p, p, p, None, p, None, p, p, p, p, p, p, need - 1,
                                 None) == EWORKSPACE
    split = shape(Nq=1, Nk=5000)                               # one row: the keys are split
    assert lib.tts_attention_workspace_bytes(split, 0) > 0
    assert lib.tts_attention_fwd(split, p, p, p, None, p, None, None, None, 0, None) == EWORKSPACE
    for empty in (shape(B=0), shape(Nq=0)):                    # nothing to do
        assert lib.tts_attention_fwd(empty, None, None, None, None, None, None, None, None, 0, None) == 0
    assert lib.tts_attention_bwd(shape(Nk=0), p, p, p, None, p, None, p, p, p, p, p, p, 1 << 40,
                                 None) == EINVAL


def test_layer_norm_refuses(lib, p):
    fwd, bwd = lib.tts_layer_norm_fwd, lib.tts_layer_norm_bwd
    assert fwd(p, 8, p, p, -1, 8, 1e-5, 0, 0, p, None, None) == EINVAL
    assert fwd(p, 8, p, p, 4, 0, 1e-5, 0, 0, p, None, None) == EINVAL
    assert fwd(p, 8, p, p, 4, 8, 1e-5, 7, 7, p, None, None) == EDTYPE
    assert fwd(p, 8, p, p, 4, 8, 1e-5, 1, 2, p, None, None) == EDTYPE   # weights of a third type
    assert fwd(None, 8, None, None, 0, 8, 1e-5, 0, 0, None, None, None) == 0
    assert bwd(p, 8, p, p, 8, p, 4, 8, 0, 0, None, None, None, None, 0, None) == EINVAL
    assert bwd(p, 8, p, p, 8, p, 4, 8, 0, 0, p, p, p, None, 0, None) == EWORKSPACE
    assert lib.tts_layer_norm_workspace_bytes(0, 8, 0) == 0
    assert lib.tts_layer_norm_workspace_bytes(1000, 64, 2) % (2 * 64 * 4) == 0


def test_embedding_refuses(lib, p):
    fwd, bwd = lib.tts_embedding_fwd, lib.tts_embedding_bwd
    assert fwd(p, 0, 8, p, 0, 4, 1.0, 0, p, None) == EINVAL
    assert fwd(p, 4, 8, p, 0, 4, 1.0, 5, p, None) == EDTYPE
    assert fwd(p, (1 << 30) + 1, 8, p, 0, 4, 1.0, 0, p, None) == ELENGTH
    assert fwd(p, 4, 8, p, 0, (1 << 30) + 1, 1.0, 0, p, None) == ELENGTH
    assert fwd(p, 4, 8, None, 0, 0, 1.0, 0, None, None) == 0
    n = lib.tts_embedding_workspace_bytes(100000, 4096, 32)
    assert n > 100000 * 8
    assert bwd(p, p, 0, 100000, 4096, 32, 1.0, 0, p, p, n - 1, None) == EWORKSPACE
    assert bwd(p, p, 0, 100000, 4096, 32, 1.0, 0, p, None, n, None) == EWORKSPACE
    assert bwd(None, p, 0, 4, 4, 8, 1.0, 0, p, p, n, None) == EINVAL


def test_wrappers_refuse_cpu_tensors():
    import torch
    from ttsplat.attention import attention
    from ttsplat.embedding import embedding
    from ttsplat.norm import layer_norm
    x = torch.zeros(1, 1, 4, 8)
    for bad in (lambda: attention(x, x, x), lambda: layer_norm(x),
                lambda: embedding(x[0, 0], torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("scale", [1e-46, 1e-39, 9e-31, 2e30])
def test_attention_refuses_scales_past_fp32(lib, p, scale):
    """1e-46 is 0 in fp32, the inverse of 1e-39 infinite: either gives NaN beside a hidden key."""
    s = shape(scale=scale)
    assert lib.tts_attention_fwd(s, p, p, p, None, p, None, None, None, 0, None) == EINVAL
    assert lib.tts_attention_bwd(s, p, p, p, None, p, None, p, p, p, p, p, p, 1 << 40, None) == EINVAL
    assert lib.tts_attention_workspace_bytes(shape(scale=1e-30), 1) > 0
    assert lib.tts_attention_workspace_bytes(shape(scale=1e30), 1) > 0

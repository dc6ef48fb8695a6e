"""What the decode-step operators around a shared prompt (qkv_norm_post, shared_prefix_attention,
adjust_logits) refuse before anything reaches a device."""
import ctypes as C

import pytest

from relay_b200 import _lib

torch = pytest.importorskip("torch")

PTR = C.c_void_p(4096)  # a 16-byte aligned address that no refused call touches
META = _lib.CTokenMeta(4096, 4096, 4096, 4096)


@pytest.fixture(autouse=True)
def no_launch():
    before = _lib.lib().rb200_kernel_launches()
    yield
    assert _lib.lib().rb200_kernel_launches() == before


def refused(rc, text):
    assert rc == -1
    with pytest.raises(ValueError, match=text):
        _lib.raise_last_error()


def qkv(**kw):
    a = dict(qkv=PTR, qkv_stride=6144, bias=None, q_norm=PTR, k_norm=PTR, eps=1e-6, inv_freq=PTR, rot=128, meta=C.byref(META), T=4,
             q_out=C.c_void_p(8192), q_stride=4096, k=PTR, v=PTR, heads=32, kv_heads=8, D=128, bs=16, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().rb200_qkv_norm_post(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(T=-1), "bad shape"), (dict(heads=0), "bad shape"), (dict(kv_heads=0), "bad shape"), (dict(bs=0), "bad shape"),
    (dict(D=127), "head_dim"), (dict(D=258, qkv_stride=1 << 20, q_stride=1 << 20), "head_dim"), (dict(D=0), "head_dim"),
    (dict(rot=3), "rot_dim"), (dict(rot=130), "rot_dim"), (dict(rot=-2), "rot_dim"),
    (dict(qkv_stride=6143), "strides"), (dict(q_stride=4095), "strides"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(qkv=None), "null"), (dict(q_out=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(meta=None), "null"),
    (dict(inv_freq=None), "null"), (dict(q_out=PTR), "same stride"),
])
def test_qkv_norm_post_refuses(kw, text):
    refused(qkv(**kw), text)


def test_qkv_norm_post_of_no_tokens_is_nothing():
    assert qkv(T=0, qkv=None, q_out=None) == 0


def prefix(shape=(32, 8, 128, 16, 6144, 4096), **kw):
    sh = _lib.CAttnShape(*shape)
    a = dict(shape=C.byref(sh), q=PTR, meta=C.byref(META), tokens=PTR, n=4, off=PTR, lens=PTR, groups=1, max_prefix=100, max_suffix=10,
             k=PTR, v=PTR, scratch=PTR, scratch_bytes=1 << 30, out=PTR, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().rb200_shared_prefix_attention(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(shape=(32, 7, 128, 16, 6144, 4096)), "head layout"), (dict(shape=(32, 8, 128, 0, 6144, 4096)), "head layout"),
    (dict(shape=(32, 8, 96, 16, 6144, 4096)), "head_dim"), (dict(shape=(32, 8, 256, 16, 12288, 8192)), "head_dim"),
    (dict(shape=(34, 2, 64, 16, 4096, 4096)), "heads/kv_heads"),
    (dict(shape=(32, 8, 128, 16, 4095, 4096)), "strides too small"), (dict(shape=(32, 8, 128, 16, 6144, 4095)), "strides too small"),
    (dict(shape=(32, 8, 128, 16, 6146, 4096)), "multiple"), (dict(shape=(32, 8, 128, 16, 6144, 4100)), "multiple"),
    (dict(n=-1), "bad batch"), (dict(n=1 << 27), "bad batch"), (dict(groups=-1), "bad batch"), (dict(max_prefix=-1), "bad batch"), (dict(max_suffix=-1), "bad batch"),
    (dict(q=None), "null"), (dict(meta=None), "null"), (dict(tokens=None), "null"), (dict(off=None), "null"), (dict(lens=None), "null"),
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(scratch=None, max_prefix=100000), "null scratch"), (dict(out=None), "null"),
    (dict(q=C.c_void_p(4104)), "aligned"), (dict(k=C.c_void_p(4098)), "aligned"), (dict(out=C.c_void_p(4104)), "aligned"),
    (dict(scratch=C.c_void_p(4100)), "aligned"), (dict(scratch_bytes=1000, max_prefix=100000), "scratch too small"),
])
def test_shared_prefix_attention_refuses(kw, text):
    refused(prefix(**kw), text)


def test_shared_prefix_attention_of_padding_only_is_nothing():
    assert prefix(n=0, q=None) == 0 and prefix(groups=0, q=None) == 0


def test_shared_prefix_scratch_is_host_computable():
    L = _lib.lib()
    sh = _lib.CAttnShape(32, 8, 128, 16, 6144, 4096)
    per = 4 * 32 * 130 * 4  # one slice of four tokens: (D + 2) floats per (token, head)
    assert L.rb200_shared_prefix_scratch_bytes(C.byref(sh), 4, 1, 100, 100) == 0  # one kernel
    assert L.rb200_shared_prefix_scratch_bytes(C.byref(sh), 4, 1, 0, 100) == 0
    for lens in ((100000, 100), (100, 100000)):
        many = L.rb200_shared_prefix_scratch_bytes(C.byref(sh), 4, 1, *lens)
        assert many > 2 * per and many % per == 0
    assert L.rb200_shared_prefix_scratch_bytes(C.byref(sh), 0, 0, 100, 100) == 0


def logits(**kw):
    a = dict(logits=PTR, ld=100, out=C.c_void_p(8192), ld_out=100, R=2, V=100, pen=PTR, history=PTR, ld_history=8, history_len=PTR,
             prompt_len=None, ids=PTR, values=PTR, ld_bias=4, bias_len=PTR, mask=PTR, ld_mask=4, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.lib().rb200_adjust_logits(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(R=-1), "bad shape"), (dict(R=65536), "bad shape"), (dict(V=0), "bad shape"), (dict(V=(1 << 30) + 1, ld=2 ** 31 - 1, ld_out=2 ** 31 - 1), "bad shape"), (dict(ld=99), "shorter"), (dict(ld_out=99), "shorter"),
    (dict(logits=None), "null"), (dict(out=None), "null"), (dict(out=PTR, ld_out=104), "same stride"),
    (dict(history=None), "history"), (dict(history_len=None), "history"), (dict(ld_history=-1), "negative"), (dict(ld_bias=-1), "negative"),
    (dict(values=None), "bias"), (dict(bias_len=None), "bias"), (dict(ld_mask=3), "mask"),
])
def test_adjust_logits_refuses(kw, text):
    refused(logits(**kw), text)


def test_the_python_wrappers_refuse_host_tensors():
    from relay_b200 import ops
    lg = torch.zeros(2, 100)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.adjust_logits(lg, lg)
    i = torch.zeros(4, dtype=torch.int32)
    meta = ops.TokenMeta(i, i, i, i)
    pool = torch.zeros(1, 1, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.qkv_norm_post(torch.zeros(4, 192), None, None, None, 1e-6, torch.zeros(32), meta, torch.zeros(4, 64), pool, pool, 1, 1, 64, 16)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.shared_prefix_attention(ops.attn_shape(1, 1, 64, 16), torch.zeros(4, 192), meta, i, i[:2], i[:1], 1, 1, pool, pool,
                                    torch.zeros(4, 64, dtype=torch.float16))

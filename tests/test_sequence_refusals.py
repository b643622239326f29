"""What the training LayerNorm and sequence attention refuse, before any launch (no GPU)."""

import ctypes

import pytest
import torch

from xfold_cpu_amd import fastnn
from xfold_cpu_amd.fastnn import config as fastnn_config
from xfold_cpu_amd.fastnn import native_hip as nh

FAKE = 1 << 40                                              # never dereferenced: the checks come first


def qkv(H=4, Hk=2, nq=6, nk=6, D=8, Dv=8, dtype=torch.float32, B=2):
    return (torch.zeros(B, H, nq, D, dtype=dtype), torch.zeros(B, Hk, nk, D, dtype=dtype),
            torch.zeros(B, Hk, nk, Dv, dtype=dtype))


@pytest.mark.parametrize("make,options,match", [
    (dict(), {}, "ROCm"),
    (dict(H=3), {}, "multiple"),
    (dict(Hk=0), {}, "multiple"),
    (dict(D=129), {}, "head dims"),
    (dict(Dv=0), {}, "head dims"),
    (dict(nq=7), {"causal": True}, "more queries"),
    (dict(nq=7), {"documents": torch.zeros(6, dtype=torch.int32)}, "more queries"),
    (dict(), {"prefix": 3}, "prefix needs"),
    (dict(), {"causal": True, "prefix": torch.zeros(2)}, "prefix must be int32"),
    (dict(), {"causal": True, "prefix": torch.zeros(3, dtype=torch.int32)}, "prefix must be int32"),
    (dict(), {"documents": torch.zeros(2, 6)}, "documents must be int32"),
    (dict(), {"documents": torch.zeros(6, dtype=torch.int64)}, "documents must be int32"),
    (dict(), {"documents": torch.zeros(5, dtype=torch.int32)}, "documents must be int32"),
    (dict(), {"lengths": torch.zeros(1, dtype=torch.int32)}, "lengths must be int32"),
    (dict(), {"slopes": torch.zeros(2)}, "slopes must be"),
    (dict(), {"slopes": torch.zeros(4, dtype=torch.float16)}, "slopes must be"),
    (dict(), {"softcap": -1.0}, "softcap"),
    (dict(), {"softcap": float("inf")}, "softcap"),
    (dict(), {"scale": float("nan")}, "scale must be finite"),
])
def test_sequence_attention_refuses(make, options, match):
    with pytest.raises(ValueError, match=match):
        fastnn.sequence_attention(*qkv(**make), **options)


def test_sequence_attention_refuses_shapes_and_backends():
    q, k, v = qkv()
    with pytest.raises(ValueError, match="do not match"):
        fastnn.sequence_attention(q, k, v[:, :, :5])
    with pytest.raises(ValueError, match="do not match"):
        fastnn.sequence_attention(q, k[:1], v)
    with pytest.raises(ValueError, match=r"\[B, H, N, D\]"):
        fastnn.sequence_attention(q[0], k, v)
    saved = fastnn_config.dot_product_attention_implementation
    try:
        fastnn_config.dot_product_attention_implementation = "torch"
        with pytest.raises(ValueError, match="only 'hip'"):
            fastnn.sequence_attention(q, k, v)
    finally:
        fastnn_config.dot_product_attention_implementation = saved


def arguments(**change):
    values = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE, lse=FAKE, dout=FAKE, dq=FAKE, dk=FAKE, dv=FAKE, batch=1, heads=4,
                  kv_heads=2, queries=8, keys=8, dim=16, value_dim=16, scale=1.0, dtype=nh.BF16)
    values.update(change)
    return nh.SequenceAttention(**values)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=7), "dtype"), (dict(dim=129), "head dims"), (dict(value_dim=0), "head dims"), (dict(kv_heads=3), "multiple"),
    (dict(kv_heads=0), "multiple"), (dict(batch=-1), "31 bits"), (dict(keys=2 ** 31), "31 bits"),
    (dict(queries=9, causal=1), "more queries"), (dict(queries=9, lengths=FAKE), "more queries"),
    (dict(prefix_all=1), "prefix"), (dict(prefix=FAKE), "prefix"), (dict(scale=float("inf")), "finite"),
    (dict(softcap=float("nan")), "finite"), (dict(softcap=1e-40), "softcap too small"), (dict(q=None), "null"), (dict(v=None), "null"), (dict(out=None), "null"),
])
def test_library_refuses(change, match):
    args = arguments(**change)
    for name in ("xfh_sequence_attention", "xfh_sequence_attention_backward"):
        with pytest.raises(ValueError, match=match):
            nh.call(name, ctypes.addressof(args), FAKE, 1 << 30, None)


def test_library_refuses_workspaces_and_missing_gradients():
    lib = nh.load_library()
    args = arguments(documents=FAKE)
    need = lib.xfh_sequence_attention_workspace_size(ctypes.addressof(args))
    assert need >= 16
    assert lib.xfh_sequence_attention(ctypes.addressof(args), FAKE, need - 1, None) == 3
    assert lib.xfh_sequence_attention(ctypes.addressof(args), None, need, None) == 3
    args = arguments()
    need = lib.xfh_sequence_attention_backward_workspace_size(ctypes.addressof(args))
    assert need >= 4 * 8 * 4
    assert lib.xfh_sequence_attention_backward(ctypes.addressof(args), FAKE, need - 1, None) == 3
    with pytest.raises(ValueError, match="null"):
        nh.call("xfh_sequence_attention_backward", ctypes.addressof(arguments(lse=None)), FAKE, 1 << 20, None)
    with pytest.raises(ValueError, match="null"):
        nh.call("xfh_sequence_attention_backward", ctypes.addressof(arguments(dk=None)), FAKE, 1 << 20, None)
    with pytest.raises(ValueError, match="no slopes"):
        nh.call("xfh_sequence_attention_backward", ctypes.addressof(arguments(dslopes=FAKE)), FAKE, 1 << 20, None)
    assert lib.xfh_sequence_attention_workspace_size(ctypes.addressof(arguments(dim=200))) == -1
    empty = arguments(batch=0)
    assert lib.xfh_sequence_attention(ctypes.addressof(empty), None, 0, None) == 0


@pytest.mark.parametrize("x,shape,w,b,eps,match", [
    (torch.zeros(3, 8), (8,), None, None, 1e-5, "ROCm"),
    (torch.zeros(3, 8, device="meta"), (8,), None, None, 1e-5, "ROCm"),
])
def test_layer_norm_refuses(x, shape, w, b, eps, match):
    with pytest.raises(ValueError, match=match):
        fastnn.trainable_layer_norm(x, shape, w, b, eps)
    with pytest.raises(ValueError, match=match):
        fastnn.LayerNorm(8)(x)


def test_layer_norm_library_refuses():
    lib = nh.load_library()
    f = ctypes.c_void_p(FAKE)
    with pytest.raises(ValueError, match="dtypes"):
        nh.call("xfh_layer_norm_train", f, 5, 4, 2, 4, None, 0, None, 0, 1e-5, f, 0, None, None)
    with pytest.raises(ValueError, match="f32 and f32"):
        nh.call("xfh_layer_norm_train", f, nh.F32, 4, 2, 4, None, 0, None, 0, 1e-5, f, nh.BF16, None, None)
    with pytest.raises(ValueError, match="stride"):
        nh.call("xfh_layer_norm_train", f, 0, 3, 2, 4, None, 0, None, 0, 1e-5, f, 0, None, None)
    with pytest.raises(ValueError, match="eps"):
        nh.call("xfh_layer_norm_train", f, 0, 4, 2, 4, None, 0, None, 0, -1.0, f, 0, None, None)
    with pytest.raises(ValueError, match="null"):
        nh.call("xfh_layer_norm_train", None, 0, 4, 2, 4, None, 0, None, 0, 1e-5, f, 0, None, None)
    with pytest.raises(ValueError, match="null"):
        nh.call("xfh_layer_norm_backward", f, 0, 4, f, 0, 4, 2, 4, None, 0, None, f, None, 0, None, 0, None, 0, None)
    need = lib.xfh_layer_norm_backward_workspace_size(1000, 64)
    assert need > 0
    assert lib.xfh_layer_norm_backward(f, 0, 64, f, 0, 64, 1000, 64, None, 0, f, f, f, 0, None, 0, f, need - 1, None) == 3
    assert lib.xfh_layer_norm_train(None, 0, 4, 0, 4, None, 0, None, 0, 1e-5, None, 0, None, None) == 0


def test_autograd_extension_of_another_abi():
    with pytest.raises(RuntimeError, match="rebuild"):
        nh.autograd().bind(nh.ABI_VERSION + 1, {})
    nh.autograd().bind(nh.ABI_VERSION, {name: ctypes.cast(nh.function(name), ctypes.c_void_p).value for name in nh.SIGNATURES})

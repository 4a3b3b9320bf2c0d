"""What the operators that serve from packed block formats refuse: shapes and types before any device is touched (no GPU needed),
through both routes to the C ABI."""
import ctypes

import pytest
import torch

import mptorch_b200.quant as q
from mptorch_b200 import _cabi
from mptorch_b200 import backend as be

U8, I32 = torch.uint8, torch.int32


@pytest.fixture(params=["ext", "ctypes"], autouse=True)
def route(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(be, "_ext", None)
    elif be._ext is None:
        pytest.skip("the extension is not built")


def weights(n=8, k=64, group=32):
    return torch.zeros(n, k // 2, dtype=U8), torch.zeros(n, k // group, dtype=U8)


def refused(match, fn, *args, **kw):
    with pytest.raises((RuntimeError, ValueError, TypeError), match=match):
        fn(*args, **kw)


def test_linear():
    c, s = weights()
    x = torch.zeros(3, 64)
    refused("CUDA", q.mx_linear, x, c, s)
    refused("float32, bfloat16 or float16", q.mx_linear, x.double(), c, s)
    refused("multiple of 32", q.mx_linear, torch.zeros(3, 48), torch.zeros(8, 24, dtype=U8), s)
    refused("codes", q.mx_linear, torch.zeros(3, 96), c, s)
    refused("scales", q.mx_linear, x, c, weights(group=16)[1])
    refused("scales", q.nvfp4_linear, x, c, s, torch.ones(1))
    refused("global_scale", q.nvfp4_linear, x, c, weights(group=16)[1], torch.ones(2))
    refused("codes", q.mx_linear, x, c.to(torch.int8), s)
    refused("codes", q.mx_linear, x, c.t().contiguous().t(), s)
    refused("bias", q.mx_linear, x, c, s, torch.zeros(7))
    refused("bias", q.mx_linear, x, c, s, torch.zeros(8, dtype=torch.bfloat16))
    refused("backward", q.mx_linear, x.requires_grad_(), c, s)


def batch(seqs=2, width=4, ragged=False):
    return (torch.zeros(seqs, width, dtype=I32), torch.ones(seqs, dtype=I32), torch.zeros(seqs + 1, dtype=I32) if ragged else None)


def test_cache_and_attention():
    cache = q.MXCache.empty(4, 2, 64, 16, device="cpu")
    p, n, st = batch()
    k = torch.zeros(2, 1, 2, 64)
    for call in (lambda *a, **kw: q.mx_cache_write(a[0], a[0], *a[1:], **kw), q.mx_attention):
        refused("CUDA", call, k, cache, p, n)
        refused("rows of 32 values", call, k[..., :32], cache, p, n)
        refused("float32, bfloat16 or float16", call, k.double(), cache, p, n)
        refused("int32", call, k, cache, p.long(), n)
        refused("int32", call, k, cache, p, n.long())
        refused("lens", call, k, cache, p, torch.ones(3, dtype=I32))
        refused("starts", call, k, cache, p, n, torch.zeros(2, dtype=I32))
        refused(r"must be \[rows", call, k, cache, p, n, torch.zeros(3, dtype=I32))
        refused(r"must be \[sequences", call, k[0], cache, p, n)
        refused(r"must be \[sequences", call, k[:1], cache, p, n)
        refused("three or four dimensions", call, k[0, 0], cache, p, n)
        refused("k_codes, k_scales", call, k, cache[:3], p, n)
        refused("k_scales|codes", call, k, (cache[1], cache[0], cache[2], cache[3]), p, n)
        refused("v_codes", call, k, (cache[0], cache[1], cache[2][:3], cache[3]), p, n)
        refused("contiguous", call, k, (cache[0].transpose(1, 2), cache[1], cache[2], cache[3]), p, n)
        refused("backward", call, k.clone().requires_grad_(), cache, p, n)
    refused("has 4 heads", q.mx_cache_write, torch.zeros(2, 1, 4, 64), torch.zeros(2, 1, 4, 64), cache, p, n)
    refused("shape and type of k", q.mx_cache_write, k, k[..., :32], cache, p, n)
    refused("shape and type of k", q.mx_cache_write, k, k.half(), cache, p, n)
    refused("do not divide", q.mx_attention, torch.zeros(2, 1, 3, 64), cache, p, n)
    refused("negative", q.mx_attention, k, cache, p, n, window=-1)
    refused("negative", q.mx_attention, k, cache, p, n, window=4, sinks=-1)
    refused("out", q.mx_attention, k, cache, p, n, out=torch.zeros(2, 1, 2, 32))
    refused("out", q.mx_attention, k, cache, p, n, out=torch.zeros(2, 1, 2, 64, dtype=torch.half))
    refused("backward", q.mx_attention, k, cache, p, n, out=torch.zeros(2, 1, 2, 64, requires_grad=True))
    refused("CUDA", q.mx_cache_read, cache, p, n, 1)
    refused("negative", q.mx_cache_read, cache, p, n, -1)


def test_empty_cache_arguments():
    refused("elem_format", q.MXCache.empty, 4, 2, 64, elem_format="e5m2", device="cpu")
    refused("head_dim", q.MXCache.empty, 4, 2, 80, device="cpu")
    refused("head_dim", q.MXCache.empty, 4, 2, 288, device="cpu")
    refused("page", q.MXCache.empty, 4, 2, 64, 48, device="cpu")
    c = q.MXCache.empty(3, 2, 96, 32, "e2m1", device="cpu")
    assert [tuple(t.shape) for t in c] == [(3, 2, 32, 48), (3, 2, 32, 3)] * 2


def test_c_abi_refuses_before_any_launch():
    """Bad descriptors, null pointers and short workspaces come back as codes with a message."""
    L = _cabi.lib()

    def err(name, *args):
        assert getattr(L, name)(*args) == 1
        return L.mpt_last_error().decode()

    one = ctypes.c_void_p(256)                      # a pointer that is checked and never followed
    assert "multiple of 32" in err("mpt_block_linear", one, one, one, None, None, one, 1, 8, 48, 0, 0, None, 0, None)
    assert "unknown format" in err("mpt_block_linear", one, one, one, None, None, one, 1, 8, 64, 7, 0, None, 0, None)
    assert "data type" in err("mpt_block_linear", one, one, one, None, None, one, 1, 8, 64, 0, 9, None, 0, None)
    assert "bad extents" in err("mpt_block_linear", one, one, one, None, None, one, -1, 8, 64, 0, 0, None, 0, None)
    assert "null pointer" in err("mpt_block_linear", None, one, one, None, None, one, 1, 8, 64, 0, 0, None, 0, None)
    assert "16 bytes" in err("mpt_block_linear", one, ctypes.c_void_p(264), one, None, None, one, 1, 8, 64, 0, 0, None, 0, None)
    assert "even address" in err("mpt_block_linear", one, one, ctypes.c_void_p(257), None, None, one, 1, 8, 64, 1, 0, None, 0, None)
    assert L.mpt_block_linear(one, one, one, None, None, one, 40, 8, 64, 0, 0, None, 0, None) == 3 and b"workspace" in L.mpt_last_error()
    assert L.mpt_block_linear(None, None, None, None, None, None, 0, 8, 64, 0, 0, None, 0, None) == 0

    def cache(**kw):
        f = dict(k_codes=256, k_scales=256, v_codes=256, v_scales=256, num_pages=4, heads=2, dim=64, page=16, elem_format=0)
        return ctypes.byref(_cabi.MxCache(**{**f, **kw}))

    def rows(**kw):
        f = dict(pages=256, lens=256, starts=None, rows=2, seqs=2, width=4)
        return ctypes.byref(_cabi.MxBatch(**{**f, **kw}))

    strides = (ctypes.c_int64 * 3)(128, 128, 64)
    att = lambda c, b, heads=2, win=0, sinks=0, q=one, out=one: err("mpt_mx_attention", c, b, q, 0, strides, heads, 1.0, win, sinks, out, 1, None, 0, None)  # noqa: E731
    for bad, text in ((dict(dim=48), "head_dim"), (dict(dim=512), "head_dim"), (dict(page=24), "page size"), (dict(page=512), "page size"),
                      (dict(elem_format=3), "element format"), (dict(heads=0), "kv heads"), (dict(num_pages=-1), "number of pages"),
                      (dict(k_codes=None), "null pointer"), (dict(v_codes=264), "16 bytes"), (dict(k_scales=260), "8 bytes"),
                      (dict(v_scales=258), "8 bytes")):
        assert text in att(cache(**bad), rows())
        assert text in err("mpt_mx_cache_write", cache(**bad), rows(), one, one, 0, strides, strides, None)
        assert text in err("mpt_mx_cache_read", cache(**bad), rows(), one, one, 0, None)
    for bad, text in ((dict(rows=3), "do not divide"), (dict(rows=-1), "bad extents"), (dict(width=1 << 28), "bad extents"), (dict(lens=None), "null pointer"),
                      (dict(pages=None), "null pointer")):
        assert text in att(cache(), rows(**bad))
    assert "null descriptor" in att(None, rows())
    assert L.mpt_mx_attention(cache(), rows(), one, 0, strides, 2, 1.0, 0, 0, one, 1, None, 0, None) == 3 and b"workspace" in L.mpt_last_error()
    assert "do not divide" in att(cache(), rows(), heads=3)
    assert "negative" in att(cache(), rows(), win=-1)
    assert "null pointer" in att(cache(), rows(), q=None)
    assert "null pointer" in err("mpt_mx_cache_write", cache(), rows(), None, one, 0, strides, strides, None)
    assert "null pointer" in err("mpt_mx_cache_read", cache(), rows(), one, None, 0, None)
    assert "data type" in err("mpt_mx_cache_read", cache(), rows(), one, one, 5, None)


def test_derivatives_are_not_dropped_in_silence():
    """Every dense input: one that needs a gradient, and a dual tensor, whose tangent no_grad does not stop."""
    import torch.autograd.forward_ad as fwd

    c, s = weights()
    nc, ns = weights(group=16)
    cache = q.MXCache.empty(4, 2, 64, 16, device="cpu")
    p, n, _ = batch()
    k, x, b, one = torch.zeros(2, 1, 2, 64), torch.zeros(3, 64), torch.zeros(8), torch.ones(1)
    calls = [(lambda t: q.mx_linear(t, c, s), x), (lambda t: q.mx_linear(x, c, s, t), b), (lambda t: q.nvfp4_linear(t, nc, ns, one), x),
             (lambda t: q.nvfp4_linear(x, nc, ns, t), one), (lambda t: q.nvfp4_linear(x, nc, ns, one, t), b),
             (lambda t: q.mx_cache_write(t, k, cache, p, n), k), (lambda t: q.mx_cache_write(k, t, cache, p, n), k),
             (lambda t: q.mx_attention(t, cache, p, n), k), (lambda t: q.mx_attention(k, cache, p, n, out=t), k.clone())]
    for call, t in calls:
        refused("backward", call, t.clone().requires_grad_())
        with torch.no_grad():
            refused("CUDA", call, t.clone().requires_grad_())
            with fwd.dual_level():
                refused("forward-mode", call, fwd.make_dual(t.clone(), torch.ones_like(t)))
            refused("CUDA", call, t)


def test_calls_in_the_readme_take_their_arguments_in_order():
    """Each call of this package in a code line of README.md fits the function, and a name that is a parameter's stands in its place."""
    import ast
    import inspect
    import os

    text = open(os.path.join(os.path.dirname(__file__), "..", "README.md")).read()
    seen = set()
    for line in text.splitlines():
        if not line.startswith("    ") or "q." not in line:
            continue
        try:
            tree = ast.parse(line.strip())
        except SyntaxError:
            continue
        for call in (n for n in ast.walk(tree) if isinstance(n, ast.Call) and isinstance(n.func, ast.Attribute)):
            fn = getattr(q, call.func.attr, None) if isinstance(call.func.value, ast.Name) and call.func.value.id == "q" else None
            if fn is None:
                continue
            seen.add(call.func.attr)
            sig = inspect.signature(fn)
            sig.bind(*call.args, **{k.arg: k.value for k in call.keywords})
            names = list(sig.parameters)
            for i, a in enumerate(call.args):
                if isinstance(a, ast.Name) and a.id in names:
                    assert names[i] == a.id, line
    assert {"mx_linear", "mx_cache_write", "mx_attention", "float_quantize", "float_mm"} <= seen

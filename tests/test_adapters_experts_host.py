"""Host-side checks of the adapter, expert-layer and gradient-clipping entry points: every refusal comes before a launch, so none
of them needs a GPU (addresses are made up and never read)."""
import ctypes as C

import pytest

from transformer_engine_amd import NVTEError
from transformer_engine_amd._lib import api, kBFloat16, kByte, kFloat8E4M3, kFloat16, kFloat32, kInt32

P = 0x1000


def lora_forward(**k):
    d = dict(x=P, a=P, b=P, ids=P, scaling=0, base=0, out=P, low=P, tokens=4, k=16, o=16, r=8, n=2, dtype=kBFloat16,
             ws=P, size=1 << 20)
    d.update(k)
    api.nvte_amd_lora_forward(*d.values(), 0)


def lora_backward(**k):
    d = dict(x=P, dy=P, a=P, b=P, ids=P, scaling=0, low=P, base_grad=0, dx=P, da=P, db=P, tokens=4, k=16, o=16, r=8, n=2,
             dtype=kBFloat16, grad_dtype=kBFloat16, ws=P, size=1 << 30)
    d.update(k)
    api.nvte_amd_lora_backward(*d.values(), 0)


@pytest.mark.parametrize("call", [lora_forward, lora_backward])
@pytest.mark.parametrize("bad", [dict(r=0), dict(r=129), dict(k=0), dict(o=0), dict(k=(1 << 24) + 1), dict(n=0), dict(dtype=kFloat32),
                                 dict(dtype=kFloat8E4M3), dict(x=0), dict(a=0), dict(b=0), dict(ids=0), dict(low=0),
                                 dict(tokens=1 << 31)])
def test_lora_refusals(call, bad):
    with pytest.raises(NVTEError):
        call(**bad)


@pytest.mark.parametrize("bad", [dict(da=0), dict(db=0), dict(n=4097, r=1), dict(grad_dtype=kFloat16), dict(ws=0), dict(size=10),
                                 dict(ws=P + 8), dict(dy=0)])
def test_lora_backward_refusals(bad):
    with pytest.raises(NVTEError):
        lora_backward(**bad)


def test_lora_forward_refuses_no_output():
    with pytest.raises(NVTEError):
        lora_forward(out=0)


@pytest.mark.parametrize("bad", [dict(ws=0), dict(size=64), dict(ws=P + 8)])
def test_lora_forward_refuses_a_bad_workspace(bad):
    assert api.nvte_amd_lora_forward_workspace_size(4, 2) == 0 < api.nvte_amd_lora_forward_workspace_size(2000, 2)
    with pytest.raises(NVTEError, match="workspace"):
        lora_forward(tokens=2000, **bad)


def test_lora_sizes():
    assert 1 <= api.nvte_amd_lora_num_slices(8192, 4096) <= 4
    assert api.nvte_amd_lora_num_slices(1 << 20, 4096) == 1
    assert 1 < api.nvte_amd_lora_num_slices(1, 4096) <= 64
    assert api.nvte_amd_lora_num_slices(0, 1) == 1
    for tokens in (0, 1, 17, 100, 5000):
        for features in (1, 63, 64, 65, 1000, 16384):
            assert 1 <= api.nvte_amd_lora_num_slices(tokens, features) <= (features + 63) // 64
    lora_forward(tokens=0, x=0, out=0, ids=0, low=0)   # nothing to do, nothing launched
    assert api.nvte_amd_lora_backward_workspace_size(8192, 4096, 4096, 16, 1) > 8192 * 16 * 4


def moe(**k):
    d = dict(x=P, w1=P, w2=P, s1=0, s2=0, ids=P, weights=P, out=P, tokens=4, top_k=2, experts=8, hidden=64, ffn=32, dtype=kBFloat16,
             wdtype=kBFloat16, ws=P, size=1 << 30)
    d.update(k)
    api.nvte_amd_moe_forward(*d.values(), 0)


@pytest.mark.parametrize("bad", [
    dict(tokens=257), dict(top_k=0), dict(top_k=65), dict(tokens=256, top_k=17), dict(experts=0), dict(experts=65536), dict(hidden=0),
    dict(ffn=0), dict(hidden=(1 << 20) + 1), dict(dtype=kFloat32), dict(dtype=kFloat32, wdtype=kFloat32), dict(wdtype=kFloat16),
    dict(wdtype=kByte), dict(s1=P), dict(s2=P), dict(wdtype=kFloat8E4M3), dict(wdtype=kFloat8E4M3, s1=P), dict(x=0), dict(w1=0),
    dict(w2=0), dict(ids=0), dict(weights=0), dict(out=0), dict(ws=0), dict(ws=P + 4), dict(size=100)])
def test_moe_refusals(bad):
    with pytest.raises(NVTEError):
        moe(**bad)


def test_moe_without_tokens():
    moe(tokens=0, x=0, out=0, ids=0, weights=0, ws=0, size=0)


@pytest.mark.parametrize("bad", [dict(experts=0), dict(experts=1025), dict(top_k=0), dict(top_k=9), dict(experts=100, top_k=65),
                                 dict(dtype=kInt32), dict(logits=0), dict(ids=0), dict(weights=0)])
def test_topk_refusals(bad):
    d = dict(logits=P, ids=P, weights=P, tokens=4, experts=8, top_k=2, renormalize=1, dtype=kFloat32)
    d.update(bad)
    with pytest.raises(NVTEError):
        api.nvte_amd_moe_topk(*d.values(), 0)


def clip(grads, outs, numels, dtypes=None, out_dtypes=None, max_norm=1.0, eps=1e-6, ws=P, size=1 << 30):
    n = len(grads)
    ptrs = lambda v: (C.c_void_p * n)(*v)
    ints = lambda v: (C.c_int * n)(*(v or [kFloat32] * n))
    api.nvte_amd_clip_grad_norm(ptrs(grads), ptrs(outs), (C.c_size_t * n)(*numels), ints(dtypes), ints(out_dtypes), n,
                                C.c_float(max_norm), C.c_float(eps), 0, ws, size, 0)


@pytest.mark.parametrize("args, text", [
    (dict(grads=[0x1000], outs=[0x1000], numels=[4], dtypes=[kInt32]), "dtype"),
    (dict(grads=[0x1000], outs=[0x2000], numels=[4], out_dtypes=[kFloat8E4M3]), "dtype"),
    (dict(grads=[0], outs=[0x1000], numels=[4]), "no data"),
    (dict(grads=[0x1000], outs=[0], numels=[4]), "no data"),
    (dict(grads=[0x1002], outs=[0x2000], numels=[4]), "aligned"),
    (dict(grads=[0x1000], outs=[0x2001], numels=[4], out_dtypes=[kFloat16]), "aligned"),
    (dict(grads=[0x1000], outs=[0x1000], numels=[4], dtypes=[kFloat16]), "dtype"),
    (dict(grads=[0x1000, 0x1000], outs=[0x1000, 0x1000], numels=[4, 4]), "overlaps"),
    (dict(grads=[0x1000, 0x2000], outs=[0x3000, 0x300c], numels=[4, 4]), "overlaps"),
    (dict(grads=[0x1000, 0x2000], outs=[0x2008, 0x4000], numels=[4, 4]), "overlaps"),
    (dict(grads=[0x2000], outs=[0x1ff8], numels=[4]), "overlaps"),
    (dict(grads=[0x1000], outs=[0x2000], numels=[4], max_norm=-1.0), "max_norm"),
    (dict(grads=[0x1000], outs=[0x2000], numels=[4], max_norm=float("nan")), "max_norm"),
    (dict(grads=[0x1000], outs=[0x2000], numels=[4], eps=float("inf")), "eps"),
    (dict(grads=[0x1000], outs=[0x2000], numels=[4], ws=0), "workspace"),
    (dict(grads=[0x1000], outs=[0x2000], numels=[4], size=8), "workspace"),
])
def test_clip_refusals(args, text):
    with pytest.raises(NVTEError, match=text):
        clip(**args)


def test_norm_workspace_grows_with_the_list():
    size = lambda *n: api.nvte_amd_grad_norm_workspace_size((C.c_size_t * len(n))(*n), len(n))
    assert size() == 8 and size(0) == 8 and size(1) == 16 and size(1, 1) == 24
    assert 2048 * 8 <= size(1 << 33) <= 2100 * 8


def test_python_wrappers_refuse_host_tensors():
    import torch

    from transformer_engine_amd.lora import lora_forward as forward
    from transformer_engine_amd.moe import moe_forward, moe_topk
    from transformer_engine_amd.weight_update import _Arrays
    bf = dict(dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU only"):
        forward(torch.zeros(2, 8, **bf), torch.zeros(1, 4, 8, **bf), torch.zeros(1, 8, 4, **bf), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU only"):
        moe_topk(torch.zeros(2, 4), 1)
    with pytest.raises(RuntimeError, match="GPU only"):
        moe_forward(torch.zeros(2, 8, **bf), torch.zeros(1, 8, 8, **bf), torch.zeros(1, 8, 4, **bf),
                    torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1))
    with pytest.raises(RuntimeError, match="GPU"):
        _Arrays([torch.zeros(3)], "grads")

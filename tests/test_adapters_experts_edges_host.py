"""Refusals at the edges of the adapter, expert and clipping entry points that need no GPU (addresses are made up and never read)."""
import ctypes as C

import pytest

from transformer_engine_amd import NVTEError
from transformer_engine_amd._lib import api, kFloat32

P = 0x1000


def _list(**k):
    d = dict(grads=(C.c_void_p * 1)(P), outs=(C.c_void_p * 1)(2 * P), numels=(C.c_size_t * 1)(4), dtypes=(C.c_int * 1)(kFloat32),
             out_dtypes=(C.c_int * 1)(kFloat32))
    d.update(k)
    return list(d.values()) + [1]


def clip(ws=P, size=1 << 20, norm=0, **k):
    api.nvte_amd_clip_grad_norm(*_list(**k), C.c_float(1.0), C.c_float(1e-6), norm, ws, size, 0)


def clip_by_sum(sum_of_squares=P, norm=0, **k):
    api.nvte_amd_clip_by_sum_of_squares(*_list(**k), sum_of_squares, C.c_float(1.0), C.c_float(1e-6), norm, 0)


def grad_norm(ws=P, size=1 << 20, total=0, norm=0, **k):
    grads, _, numels, dtypes, _, n = _list(**k)
    api.nvte_amd_grad_norm(grads, numels, dtypes, n, total, norm, ws, size, 0)


@pytest.mark.parametrize("missing", ["grads", "outs", "numels", "dtypes", "out_dtypes"])
@pytest.mark.parametrize("call", [clip, clip_by_sum])
def test_clipping_refuses_missing_lists(call, missing):
    with pytest.raises(NVTEError, match="NULL"):
        call(**{missing: 0})


@pytest.mark.parametrize("missing", ["grads", "numels", "dtypes"])
def test_norm_refuses_missing_lists(missing):
    with pytest.raises(NVTEError, match="NULL"):
        grad_norm(**{missing: 0})


@pytest.mark.parametrize("call, bad", [(clip, dict(ws=P + 4)), (grad_norm, dict(ws=P + 4)), (clip_by_sum, dict(sum_of_squares=P + 4)),
                                       (grad_norm, dict(total=P + 4)), (clip, dict(norm=P + 2)), (grad_norm, dict(norm=P + 2)),
                                       (clip_by_sum, dict(norm=P + 2))])
def test_clipping_refuses_misaligned_sums(call, bad):
    with pytest.raises(NVTEError, match="aligned"):
        call(**bad)


@pytest.mark.parametrize("tokens, k, o, rank, n", [(4096, 4096, 14336, 64, 4096), (8, 4096, 14336, 16, 512), (600, 64, 96, 128, 7),
                                                   (64, 2056, 2731, 20, 9000), (8192, 4096, 4096, 16, 1)])
def test_a_pass_without_weight_gradients_needs_no_space_for_them(tokens, k, o, rank, n):
    size = api.nvte_amd_lora_dgrad_workspace_size(tokens, o, rank, n)
    rank_vectors = api.nvte_amd_lora_num_slices(tokens, o) * tokens * rank * 4
    lists = (tokens + 32 * (n + 1)) * 5 + 1024       # every adapter's tokens in blocks of 32, and each block's adapter
    assert 0 < size <= rank_vectors + n * rank * o * 2 + lists + 5 * 256
    if n <= 4096:
        assert size < api.nvte_amd_lora_backward_workspace_size(tokens, k, o, rank, n)


def _backward(ws, size, da=P, db=P, tokens=8, n=512):
    api.nvte_amd_lora_backward(P, P, P, P, P, 0, P, 0, P, da, db, tokens, 4096, 14336, 16, n, 6, 6, ws, size, 0)


def test_workspace_of_a_pass_without_weight_gradients_is_checked_by_its_own_size():
    small, large = api.nvte_amd_lora_dgrad_workspace_size(8, 14336, 16, 512), \
        api.nvte_amd_lora_backward_workspace_size(8, 4096, 14336, 16, 512)
    for bad in (dict(ws=P, size=small - 1, da=0, db=0), dict(ws=0, size=small, da=0, db=0), dict(ws=P, size=small),
                dict(ws=P, size=large - 1)):
        with pytest.raises(NVTEError, match="workspace of"):
            _backward(**bad)
    assert api.nvte_amd_lora_dgrad_workspace_size(0, 14336, 16, 512) == 0
    _backward(0, 0, da=0, db=0, tokens=0)               # nothing to do, nothing launched


def test_router_refuses_more_tokens_than_a_launch_has_threads_for():
    for tokens in ((1 << 26) - 3, 1 << 26, 1 << 40):
        with pytest.raises(NVTEError, match="too many tokens"):
            api.nvte_amd_moe_topk(P, P, P, tokens, 8, 2, 1, kFloat32, 0)


def test_batches_are_put_in_order_only_where_their_pool_is_small_beside_them():
    size = api.nvte_amd_lora_forward_workspace_size
    for tokens, adapters in ((511, 2), (512, 1), (512, 257), (512, 4096), (1024, 1024), (8191, 4096), (1 << 20, 4097)):
        assert size(tokens, adapters) == 0, (tokens, adapters)
    for tokens, adapters in ((512, 2), (512, 256), (2048, 1024), (8192, 4096)):
        assert size(tokens, adapters) > tokens * 4, (tokens, adapters)

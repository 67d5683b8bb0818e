"""Adapters, experts and clipping at the edges of what their entry points allow: memory, gradients that must not get lost, calls at
once, the largest sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import test_lora_gpu as lora_tests
    import test_moe_gpu as moe_tests
    from transformer_engine_amd import NVTEError
    from transformer_engine_amd._lib import api, kBFloat16
    from transformer_engine_amd.linear import linear_backward, linear_forward
    from transformer_engine_amd.lora import LoRALinear, lora, lora_backward, lora_forward
    from transformer_engine_amd.moe import moe_forward, moe_topk
    from transformer_engine_amd.recipe import DelayedScaling, Float8CurrentScaling, MXFP8BlockScaling
    from transformer_engine_amd.tensor import current_stream_ptr
    from transformer_engine_amd.weight_update import clip_grad_norm, grad_norm


@pytest.mark.parametrize("t, n", [(3, 5), (40, 300), (700, 6), (700, 1), (520, 5000)])
def test_activation_gradients_alone_stay_in_their_own_workspace(t, n):
    k, o, r = 136, 264, 24
    x, a, b, ids, s, _, dy, gbase = lora_tests.make(t, k, o, r, n, torch.bfloat16, seed=t + n)
    want = lora_tests.oracle(x, a, b, ids, s, None, dy, gbase)
    size = api.nvte_amd_lora_dgrad_workspace_size(t, o, r, n)
    ws = torch.full((size + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    dx = torch.empty_like(x)
    api.nvte_amd_lora_backward(x.data_ptr(), dy.data_ptr(), a.data_ptr(), b.data_ptr(), ids.data_ptr(), s.data_ptr(), x.data_ptr(),
                               gbase.data_ptr(), dx.data_ptr(), 0, 0, t, k, o, r, n, kBFloat16, kBFloat16, ws.data_ptr(), size,
                               current_stream_ptr())     # `low` is not read without weight gradients
    assert (ws[size:] == 0xA5).all()
    lora_tests.check("dx", dx, want[0]["dx"], want[1]["dx"], o + r + 2)
    _, saved = lora_forward(x, a, b, ids, s)
    assert torch.equal(lora_backward(dy, saved, base_grad=gbase, requires_wgrad=False)[0], dx)
    if n <= 4096:
        assert torch.equal(lora_backward(dy, saved, base_grad=gbase)[0], dx)


def test_activation_gradients_alone_take_little_memory():
    t, k, o, r, n = 64, 2048, 4096, 16, 512
    x, a, b, ids, s, _, dy, _ = lora_tests.make(t, k, o, r, n, torch.bfloat16, std=0.1)
    _, saved = lora_forward(x, a, b, ids, s)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    lora_backward(dy, saved, requires_wgrad=False)
    taken = torch.cuda.max_memory_allocated() - before
    # B transposed, partial rank vectors and dx; weight gradients' partial sums alone would be 64 * 16 * (2048 + 4096) * 4 = 25 MB
    assert taken <= b.numel() * 2 + 2 * t * k + 64 * t * r * 4 + (2 << 20), taken


def _penalty(f, at):
    """f and the sum of its gradient's squares, as a gradient penalty adds them."""
    y = f()
    g, = torch.autograd.grad(y.float().sum(), (at,), create_graph=True)
    return y.float().sum() + g.float().square().sum()


@pytest.mark.parametrize("which", [0, 1, 2])
def test_second_derivatives_of_adapters_raise(which):
    x, a, b, ids, s, base, _, _ = lora_tests.make(20, 64, 96, 8, 3, torch.bfloat16)
    args = [v.requires_grad_() for v in (x, a, b)]
    loss = _penalty(lambda: lora(*args, ids, s, base), args[which])
    with pytest.raises(RuntimeError, match="second derivatives"):
        loss.backward()


def test_first_derivatives_and_the_projections_own_chain_go_on():
    x, a, b, ids, s, base, dy, _ = lora_tests.make(20, 64, 96, 8, 3, torch.bfloat16)
    x, a, b, base = (v.requires_grad_() for v in (x, a, b, base))
    lora(x, a, b, ids, s, base).backward(dy)
    assert not any(v.grad.requires_grad for v in (x, a, b, base))
    want = [v.grad.clone() for v in (x, a, b, base)]
    got = torch.autograd.grad(lora(x, a, b, ids, s, base), (x, a, b, base), dy, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    scale = torch.ones((), device="cuda", dtype=torch.bfloat16, requires_grad=True)   # dy reaches base unchanged, any number of times
    g, = torch.autograd.grad(lora(x, a, b, ids, s, base), (base,), dy * scale, create_graph=True)
    g.float().sum().backward(inputs=[scale])
    want = dy.float().sum()
    assert abs(scale.grad.float() - want) <= 2.0 ** -8 * dy.float().abs().sum()   # dy * scale, its gradient's sum and result in bf16


def test_second_derivatives_of_the_module_raise():
    m = LoRALinear(64, 96, rank=8)
    x = torch.randn(32, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    for at in (x, m.lora_a, m.lora_b):
        with pytest.raises(RuntimeError, match="second derivatives"):
            _penalty(lambda: m(x), at).backward()


def test_a_projection_that_is_trained_is_refused():
    m = LoRALinear(64, 96, rank=8)
    x = torch.randn(32, 64, device="cuda", dtype=torch.bfloat16)
    for p in (m.linear.weight, m.linear.bias):
        p.requires_grad_()
        with pytest.raises(RuntimeError, match="frozen"):
            m(x)
        with torch.no_grad():
            assert torch.isfinite(m(x).float()).all()
        p.requires_grad_(False)
    m(x).float().sum().backward()
    assert m.lora_b.grad is not None


def test_a_scaling_that_is_trained_is_refused():
    x, a, b, ids, s, base, _, _ = lora_tests.make(20, 64, 96, 8, 3, torch.bfloat16)
    s.requires_grad_()
    with pytest.raises(RuntimeError, match="scaling"):
        lora(x, a, b, ids, s, base)
    with torch.no_grad():
        lora(x, a, b, ids, s, base)


def test_expert_layers_do_not_lose_gradients():
    x, w1, w2, ids, weights, _, _ = moe_tests.make(5, 64, 48, 4, 2, torch.bfloat16)
    plain = moe_forward(x, w1, w2, ids, weights)
    assert not plain.requires_grad
    for i in (0, 1, 2, 4):
        args = [v.clone() for v in (x, w1, w2, ids, weights)]
        args[i].requires_grad_()
        out = moe_forward(*args)
        assert torch.equal(out, plain)
        with pytest.raises(RuntimeError, match="GroupedLinear"):
            out.float().sum().backward()
        with torch.no_grad():
            assert not moe_forward(*args).requires_grad
    logits = torch.randn(5, 4, device="cuda")
    want = moe_topk(logits, 2)
    top, w = moe_topk(logits.clone().requires_grad_(), 2)
    assert torch.equal(top, want[0]) and torch.equal(w, want[1]) and not top.requires_grad
    with pytest.raises(RuntimeError, match="moe_topk"):
        w.sum().backward()


@pytest.mark.parametrize("recipe", ["delayed", "current", "mxfp8"])
def test_a_frozen_projection_holds_nothing_that_backward_does_not_read(recipe):
    rec = {"delayed": DelayedScaling, "current": Float8CurrentScaling, "mxfp8": MXFP8BlockScaling}[recipe]
    t, k, o, r = 4096, 2048, 1024, 8
    m = LoRALinear(k, o, rank=r, recipe=rec())
    torch.nn.init.normal_(m.lora_b, std=0.1)
    ids = torch.zeros(t, dtype=torch.int32, device="cuda")
    for needs_dx in (True, False):
        x = torch.randn(t, k, device="cuda", dtype=torch.bfloat16, requires_grad=needs_dx)
        m(x, ids)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = m(x, ids)
        held = torch.cuda.memory_allocated() - before
        # y, the partial rank vectors and, where dx is wanted, the weight's FP8 copies; x's would add t * k = 8 MB
        weight = (2 * k * o + k * o // 8) * needs_dx
        low = api.nvte_amd_lora_num_slices(t, k) * t * r * 4
        assert held <= 2 * t * o + low + weight + (1 << 20), (held, weight)
        dy = torch.randn_like(y)
        y.backward(dy)
        assert (x.grad is not None) == needs_dx and m.lora_a.grad is not None


@pytest.mark.parametrize("recipe", ["current", "mxfp8"])
def test_gradients_beside_a_frozen_projection_are_the_bare_passes(recipe):
    rec = {"current": Float8CurrentScaling, "mxfp8": MXFP8BlockScaling}[recipe]
    m = LoRALinear(256, 384, rank=8, num_adapters=3, recipe=rec())
    torch.nn.init.normal_(m.lora_b, std=0.1)
    x = torch.randn(64, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ids = torch.randint(-1, 3, (64,), device="cuda", dtype=torch.int32)
    y = m(x, ids)
    dy = torch.randn_like(y)
    y.backward(dy)
    with torch.no_grad():
        base, q = linear_forward(x, m.linear.weight, m.linear.bias, m.linear.fp8_state)
        want, saved = lora_forward(x, m.lora_a, m.lora_b, ids, m.scaling, base=base)
        base_grad, _, _ = linear_backward(dy, q, m.linear.fp8_state)
        dx, da, db = lora_backward(dy, saved, base_grad=base_grad)
    for got, w in ((y, want), (x.grad, dx), (m.lora_a.grad, da), (m.lora_b.grad, db)):
        assert torch.equal(got, w)


def test_casting_a_module_keeps_the_scaling_exact():
    m = LoRALinear(64, 96, rank=20, alpha=16.0, num_adapters=2)          # 0.8: not a bf16 value
    x = torch.randn(32, 64, device="cuda", dtype=torch.bfloat16)
    ids = torch.randint(-1, 2, (32,), device="cuda", dtype=torch.int32)
    torch.nn.init.normal_(m.lora_b)
    want = m(x, ids)
    for cast in (lambda: m.to(torch.bfloat16), m.bfloat16, lambda: torch.nn.Sequential(m).to("cuda", torch.bfloat16)):
        cast()
        assert m.scaling.dtype == torch.float32 and (m.scaling == torch.tensor(0.8)).all()
    assert m.state_dict()["scaling"].dtype == torch.float32
    got = m(x, ids)
    assert got.dtype == want.dtype and torch.isfinite(got.float()).all()
    m.half()
    assert m.scaling.dtype == torch.float32 and m(x.half(), ids).dtype == torch.float16


def test_many_adapters_beside_a_wide_projection():
    """More matrices to transpose than one launch has workgroups for."""
    t, k, o, r, n = 5, 16, 65536, 1, 4096
    x, a, b, _, s, _, dy, _ = lora_tests.make(t, k, o, r, n, torch.bfloat16)
    ids = torch.tensor([0, 4095, -1, 2048, 4095], dtype=torch.int32, device="cuda")
    y, saved = lora_forward(x, a, b, ids, s)
    dx, da, db = lora_backward(dy, saved)
    assert torch.equal(lora_backward(dy, saved, requires_wgrad=False)[0], dx)
    used = [0, 2048, 4095]
    few = torch.tensor([0, 2, -1, 1, 2], device="cuda")
    lora_tests.check_all((x, a[used], b[used], few, s[used], None, dy, None), y, dx, da[used], db[used])
    for grad in (da, db):
        assert (grad.flatten(1).abs().sum(1) > 0).nonzero().flatten().tolist() == used


def test_the_largest_number_of_tokens():
    t, k, o, r = 1 << 27, 4, 8, 1
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(t, k, generator=g, device="cuda", dtype=torch.bfloat16)
    dy = torch.randn(t, o, generator=g, device="cuda", dtype=torch.bfloat16)
    a, b = torch.randn(1, r, k, device="cuda", dtype=torch.bfloat16), torch.randn(1, o, r, device="cuda", dtype=torch.bfloat16)
    ids = torch.full((t,), -1, dtype=torch.int32, device="cuda")
    rows = torch.cat([torch.arange(100, device="cuda"), torch.randint(0, t, (800,), generator=g, device="cuda"),
                      torch.arange(t - 100, t, device="cuda")]).unique()
    ids[rows] = 0
    y, saved = lora_forward(x, a, b, ids)
    dx, da, db = lora_backward(dy, saved)
    one = torch.zeros(len(rows), dtype=torch.int32, device="cuda")
    lora_tests.check_all((x[rows], a, b, one, None, None, dy[rows], None), y[rows], dx[rows], da, db)
    for v in (y, dx):
        v[rows] = 0
        assert v.count_nonzero() == 0
    with pytest.raises(NVTEError, match="tokens"):
        lora_forward(torch.cat([x, x[:1]]), a, b, torch.cat([ids, ids[:1]]))


def _work(seed):
    """One user's module, requests, experts and gradients, unlike another's, and a step through all of them: decode of 33 tokens, a training
    batch long enough to be ordered by adapter, clipping."""
    torch.manual_seed(seed)
    m = LoRALinear(256, 192, rank=8, num_adapters=4, recipe=Float8CurrentScaling())
    torch.nn.init.normal_(m.lora_b, std=0.1)
    x = torch.randn(33, 256, device="cuda", dtype=torch.bfloat16)
    ids = torch.randint(-1, 4, (33,), device="cuda", dtype=torch.int32)
    router = torch.randn(192, 16, device="cuda") * 192 ** -0.5
    _, w1, w2, _, _, s1, s2 = moe_tests.make(1, 192, 136, 16, 2, torch.bfloat16, fp8=True, seed=seed)
    xt, a, b, it, s, base, dy, gbase = lora_tests.make(1400, 264, 392, 16, 5, torch.bfloat16, seed=seed)
    outs = [torch.empty_like(v, dtype=torch.float32) for v in (a, b)]
    def step():
        with torch.no_grad():
            h = m(x, ids)
        top, weights = moe_topk(h.float() @ router, 2)
        out = moe_forward(h, w1, w2, top, weights, s1, s2)
        y, saved = lora_forward(xt, a, b, it, s, base=base)
        dx, da, db = lora_backward(dy, saved, base_grad=gbase)
        few = lora_backward(dy, saved, requires_wgrad=False)[0]
        norm = clip_grad_norm([da, db], 1.0, outs=outs)
        return [v.clone() for v in (h, top, weights, out, y, dx, da, db, few, norm, *outs)]
    return step


def test_two_users_on_two_streams():
    steps = [_work(1), _work(2)]
    want = [step() for step in steps]
    torch.cuda.synchronize()
    assert not any(torch.equal(p, q) for p, q in zip(*want))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(8):
        for s, step, g in zip(streams, steps, got):
            with torch.cuda.stream(s):
                g.append(step())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for outs in g:
            assert all(torch.equal(p, q) for p, q in zip(outs, w))


def test_two_users_in_two_graphs_at_once():
    steps = [_work(3), _work(4)]
    want = [step() for step in steps]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, held = [], []
    for step, s in zip(steps, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step())
    torch.cuda.synchronize()
    for _ in range(5):
        for outs in held:
            for v in outs:
                v.zero_()
        steps[0]()                                   # a third user between the replays
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for outs, w in zip(held, want):
            assert all(torch.equal(p, q) for p, q in zip(outs, w))


def _rank_grads(rank):
    """Every rank another list: lengths, dtypes and sizes of its own, the last rank none at all."""
    g = torch.Generator(device="cuda").manual_seed(100 + rank)
    lengths, std = ([5000, 17], [40_001, 1, 333], [])[rank], (1.0, 30.0, 0.0)[rank]
    return [(torch.randn(n, generator=g, device="cuda") * std).to((torch.bfloat16, torch.float32)[(i + rank) % 2])
            for i, n in enumerate(lengths)]


def _clip_over_ranks(rank, world, port, ret):
    import os
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        torch.cuda.set_device(0)
        everyone = [v.double().square().sum().item() for r in range(world) for v in _rank_grads(r)]
        want = sum(everyone) ** 0.5
        grads = _rank_grads(rank)
        keep = [v.clone() for v in grads]
        assert abs(grad_norm(grads, group=dist.group.WORLD).item() - want) <= want * 2.0 ** -23
        for outs in ([torch.empty_like(v, dtype=torch.float32) for v in grads], None):
            norm = clip_grad_norm(grads, 2.0, outs=outs, group=dist.group.WORLD)
            assert norm.shape == (1,) and abs(norm.item() - want) <= want * 2.0 ** -23
            for k, o in zip(keep, grads if outs is None else outs):
                exact = k.double() * (2.0 / (want + 1e-6))
                assert ((o.double() - exact).abs() <= exact.abs() * (torch.finfo(o.dtype).eps / 2 + 2.0 ** -22) + 1e-38).all()
        bits = torch.tensor([norm.item()], dtype=torch.float64)
        low, high = bits.clone(), bits.clone()
        dist.all_reduce(low, op=dist.ReduceOp.MIN)
        dist.all_reduce(high, op=dist.ReduceOp.MAX)
        assert low == high == bits
        ret[rank] = "ok"
    except Exception:
        import traceback
        ret[rank] = traceback.format_exc()
    finally:
        dist.destroy_process_group()


def test_norm_and_clip_over_three_ranks():
    import socket
    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ret = mp.get_context("spawn").Manager().dict()
    mp.spawn(_clip_over_ranks, args=(3, port, ret), nprocs=3, join=True)
    assert dict(ret) == {0: "ok", 1: "ok", 2: "ok"}, dict(ret)


@pytest.mark.parametrize("ids", ["mixed", "runs"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,o,r,n", [(512, 136, 264, 16, 400), (1500, 72, 104, 40, 1000), (5000, 264, 136, 16, 3000), (4100, 7, 12, 5, 4096)])
def test_many_adapters_for_the_tokens_at_hand(t, k, o, r, n, dtype, ids):
    x, a, b, i, s, base, dy, gbase = lora_tests.make(t, k, o, r, n, dtype, seed=t, ids=ids, std=0.5)
    y, saved = lora_forward(x, a, b, i, s, base=base)
    dx, da, db = lora_backward(dy, saved, base_grad=gbase)
    lora_tests.check_all((x, a, b, i, s, base, dy, gbase), y, dx, da, db)
    alone = lora_backward(dy, saved, base_grad=gbase, requires_wgrad=False)[0]
    lora_tests.check_all((x, a, b, i, s, base, dy, gbase), y, alone, da, db)

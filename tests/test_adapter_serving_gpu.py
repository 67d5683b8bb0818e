"""Adapters, the expert layer and gradient clipping together, as a fine-tuning step and as a decode step use them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    import test_lora_gpu as lora_tests
    import test_moe_gpu as moe_tests
    from transformer_engine_amd.lora import LoRALinear
    from transformer_engine_amd.moe import moe_forward, moe_topk
    from transformer_engine_amd.normalization import rmsnorm_fwd
    from transformer_engine_amd.recipe import Float8CurrentScaling, MXFP8BlockScaling
    from transformer_engine_amd.weight_update import clip_grad_norm, grad_norm


def _recipes():
    return {"current": Float8CurrentScaling(), "mxfp8": MXFP8BlockScaling()}


@pytest.mark.parametrize("recipe", ["delayed", "current", "mxfp8"])
def test_fine_tuning_step(recipe):
    """Two frozen FP8 projections with adapters, ragged requests, clipped gradients in fp32, one step of descent."""
    torch.manual_seed(1)
    rec = None if recipe == "delayed" else _recipes()[recipe]
    up = LoRALinear(256, 512, rank=8, num_adapters=4, alpha=16.0, recipe=rec)
    down = LoRALinear(512, 256, rank=8, num_adapters=4, alpha=16.0, recipe=rec)
    for m in (up, down):
        torch.nn.init.normal_(m.lora_b, std=0.1)
    x = torch.randn(640, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ids = torch.randint(-1, 4, (640,), device="cuda", dtype=torch.int32)
    keep = {}
    h = up(x, ids)
    h.retain_grad()
    act = torch.nn.functional.silu(h)
    act.retain_grad()
    y = down(act, ids)
    dy = torch.randn_like(y) * 0.1
    y.backward(dy)
    # the adapters' gradients of the last projection have no FP8 in them: x, dy and the pools are what the formula reads
    val, mag = lora_tests.oracle(act.detach(), down.lora_a.detach(), down.lora_b.detach(), ids, down.scaling, None, dy, None)
    lora_tests.check("da", down.lora_a.grad, val["da"], mag["da"], 256 + 640 + 2)
    lora_tests.check("db", down.lora_b.grad, val["db"], mag["db"], 512 + 640 + 2)
    val, mag = lora_tests.oracle(x.detach(), up.lora_a.detach(), up.lora_b.detach(), ids, up.scaling, None, h.grad, None)
    lora_tests.check("da", up.lora_a.grad, val["da"], mag["da"], 512 + 640 + 2)
    params = [up.lora_a, up.lora_b, down.lora_a, down.lora_b]
    assert up.linear.weight.grad is None and torch.isfinite(x.grad.float()).all()
    grads = [p.grad for p in params]
    clipped = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    limit = grad_norm(grads).item() / 2
    norm = clip_grad_norm(grads, limit, outs=clipped)
    assert abs(grad_norm(clipped).item() - limit) <= limit * 1e-5 and norm.item() == grad_norm(grads).item()
    with torch.no_grad():
        for p, g in zip(params, clipped):
            keep[p] = p.clone()
            p -= 0.5 * g
    assert all(not torch.equal(p, keep[p]) for p in params)


def _decode_parts():
    torch.manual_seed(2)
    hidden, ffn, experts = 256, 192, 8
    norm_w = torch.rand(hidden, device="cuda", dtype=torch.bfloat16) + 0.5
    proj = LoRALinear(hidden, hidden, rank=16, num_adapters=5, recipe=Float8CurrentScaling())
    torch.nn.init.normal_(proj.lora_b, std=0.1)
    router = torch.randn(hidden, experts, device="cuda") * hidden ** -0.5
    _, w1, w2, _, _, s1, s2 = moe_tests.make(1, hidden, ffn, experts, 2, torch.bfloat16, fp8=True, seed=3)
    def step(x, ids):
        n, _, _ = rmsnorm_fwd(x, norm_w, 1e-5)
        h = proj(n, ids)
        top, weights = moe_topk(h.float() @ router, 2)
        return n, h, top, weights, moe_forward(h, w1, w2, top, weights, s1, s2)
    return step, proj, (w1, w2, s1, s2), router


@pytest.mark.parametrize("tokens", [1, 7, 64])
def test_decode_step(tokens):
    step, proj, (w1, w2, s1, s2), router = _decode_parts()
    x = torch.randn(tokens, 256, device="cuda", dtype=torch.bfloat16)
    ids = torch.randint(-1, 5, (tokens,), device="cuda", dtype=torch.int32)
    with torch.no_grad():
        n, h, top, weights, out = step(x, ids)
        base = proj.linear(n)                       # the same FP8 product without adapters
        val, mag = lora_tests.oracle(n, proj.lora_a, proj.lora_b, ids, proj.scaling, base, base, None)
        lora_tests.check("h", h, val["y"], mag["y"], 256 + 16 + 2)
        assert torch.equal(h[ids < 0], base[ids < 0])
        assert torch.equal(top.long(), (h.float() @ router).sort(dim=-1, descending=True, stable=True).indices[:, :2])
        moe_tests.check(out, (h, w1, w2, top, weights, s1, s2))


def test_decode_steps_captured_with_new_requests():
    step, _, _, _ = _decode_parts()
    x = torch.randn(12, 256, device="cuda", dtype=torch.bfloat16)
    ids = torch.randint(-1, 5, (12,), device="cuda", dtype=torch.int32)
    with torch.no_grad():
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(x, ids)
        torch.cuda.current_stream().wait_stream(stream)
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(x, ids)
        with torch.cuda.graph(other):
            held2 = step(x, ids)
        for _ in range(4):
            x.copy_(torch.randn(12, 256, device="cuda"))
            ids.copy_(torch.randint(-1, 5, (12,), device="cuda"))
            eager = [v.clone() for v in step(x, ids)]
            torch.cuda.synchronize()
            graph.replay()
            other.replay()
            graph.replay()
            torch.cuda.synchronize()
            for got in (held, held2):
                assert all(torch.equal(p, q) for p, q in zip(got, eager))


def test_two_streams_at_once():
    """The same calls on two streams, nothing shared between them but the inputs."""
    step, _, _, _ = _decode_parts()
    x = torch.randn(64, 256, device="cuda", dtype=torch.bfloat16)
    ids = torch.randint(-1, 5, (64,), device="cuda", dtype=torch.int32)
    with torch.no_grad():
        want = step(x, ids)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        got = [[], []]
        for _ in range(5):
            for s, g in zip(streams, got):
                with torch.cuda.stream(s):
                    g.append(step(x, ids))
        torch.cuda.synchronize()
    for g in got:
        for outs in g:
            assert all(torch.equal(p, q) for p, q in zip(outs, want))

"""Global gradient norm and clipping against 64-bit sums.

Bounds: squares are summed in 64 bits, so the norm is off by its one rounding to fp32 (half a step, 2^-24) and a few 2^-53; the
factor is rounded to fp32 once (2^-24), the product once in fp32 (2^-24) and once to the output's type (half a step)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from transformer_engine_amd.weight_update import clip_grad_norm, grad_norm

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(lengths, dtypes, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * std).to(dtypes[i % len(dtypes)]) for i, n in enumerate(lengths)]


def norm64(grads):
    return torch.stack([g.double().square().sum() for g in grads] + [torch.zeros((), dtype=torch.float64, device="cuda")]).sum().sqrt()


def check(grads, outs, norm, max_norm, eps=1e-6):
    n = norm64(grads)
    assert norm.shape == (1,) and norm.dtype == torch.float32
    assert abs(norm.item() - n.item()) <= n.item() * (2.0 ** -24 + 2.0 ** -45)
    c = min(1.0, max_norm / (n.item() + eps))
    for g, o in zip(grads, outs):
        want = g.double() * c
        info = torch.finfo(o.dtype)
        bound = want.abs() * (info.eps / 2 + 2.0 ** -22) + info.smallest_normal * info.eps
        assert ((o.double() - want).abs() <= bound).all()


LISTS = [[1], [7, 1, 16384, 16385], [3, 100000, 5], [65536] * 20, [1] * 300, [200_003, 17, 1_000_001, 32768]]


@pytest.mark.parametrize("dtypes", [[d] for d in DTYPES] + [DTYPES])
@pytest.mark.parametrize("lengths", LISTS, ids=[str(i) for i in range(len(LISTS))])
def test_norm_and_clip(lengths, dtypes):
    grads = make(lengths, dtypes, seed=len(lengths))
    keep = [g.clone() for g in grads]
    n = norm64(grads).item()
    assert abs(grad_norm(grads).item() - n) <= n * (2.0 ** -24 + 2.0 ** -45)
    for out_dtype in DTYPES:
        outs = [torch.full((g.numel(),), float("nan"), dtype=out_dtype, device="cuda") for g in grads]
        check(keep, outs, clip_grad_norm(grads, 0.5 * n, outs=outs), 0.5 * n)
        assert all(torch.equal(g, k) for g, k in zip(grads, keep))
    check(keep, grads, clip_grad_norm(grads, 0.25 * n), 0.25 * n)


def test_nothing_changes_below_the_limit():
    grads = make([5, 40000], DTYPES[1:], std=1e-3)
    keep = [g.clone() for g in grads]
    clip_grad_norm(grads, 1e4)
    assert all(torch.equal(g, k) for g, k in zip(grads, keep))
    outs = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    clip_grad_norm(grads, float("inf"), outs=outs)
    assert all(torch.equal(o, k.float()) for o, k in zip(outs, keep))
    clip_grad_norm(grads, 0.0)
    assert all((g == 0).all() for g in grads)


def test_squares_neither_overflow_nor_vanish():
    for value in (1e30, 1e-30):
        grads = [torch.full((1000,), value, device="cuda"), torch.full((24,), value, device="cuda", dtype=torch.bfloat16)]
        n = norm64(grads).item()
        assert abs(grad_norm(grads).item() - n) <= n * 2.0 ** -23


def test_inf_and_nan_reach_the_norm():
    grads = make([100, 3000], [torch.float32])
    grads[1][7] = float("inf")
    norm = clip_grad_norm(grads, 1.0)
    assert norm.item() == float("inf") and grads[1][7].isnan() and (grads[0] == 0).all()
    grads = make([100, 3000], [torch.bfloat16])
    grads[0][99] = float("nan")
    norm = clip_grad_norm(grads, 1.0)
    assert norm.isnan().all() and all(g.isnan().all() for g in grads)


@pytest.mark.parametrize("out_off", [0, 1, 3])
@pytest.mark.parametrize("off", [0, 1, 5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_a_flat_buffer_leave_their_neighbours_alone(dtype, off, out_off):
    lengths = [1, 33, 5000, 16384, 40001]
    total = sum(lengths) + 7 * len(lengths) + off
    g = torch.Generator(device="cuda").manual_seed(off)
    flat = torch.randn(total, generator=g, device="cuda").to(dtype)
    dest = torch.full((total + 8,), 5.0, dtype=torch.float32, device="cuda")
    grads, outs, at, used = [], [], off, torch.zeros(total + 8, dtype=torch.bool, device="cuda")
    for n in lengths:
        grads.append(flat[at:at + n])
        outs.append(dest[at + out_off:at + out_off + n])
        used[at + out_off:at + out_off + n] = True
        at += n + 7
    check(grads, outs, clip_grad_norm(grads, 1.0, outs=outs), 1.0)
    assert (dest[~used] == 5.0).all()
    before = flat.clone()
    norm = clip_grad_norm(grads, 1.0)
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for v in grads:
        inside[(v.data_ptr() - flat.data_ptr()) // flat.element_size():][:v.numel()] = True
    assert torch.equal(flat[~inside], before[~inside]) and norm.item() > 1


def test_empty_tensors_and_empty_lists():
    e = torch.empty(0, device="cuda")
    assert grad_norm([]).item() == 0 and grad_norm([e]).item() == 0 and clip_grad_norm([e, e], 1.0).item() == 0
    grads = [e, torch.full((4,), 3.0, device="cuda"), torch.empty(0, device="cuda", dtype=torch.bfloat16)]
    assert clip_grad_norm(grads, 3.0, eps=0.0).item() == 6.0 and (grads[1] == 1.5).all()


def test_the_same_bits_every_time_and_for_any_split_of_the_work():
    grads = make([3_000_001, 17, 90_000], DTYPES, seed=5)
    norms = {grad_norm(grads).item() for _ in range(5)}
    outs = [torch.empty_like(g) for g in grads]
    norms |= {clip_grad_norm(grads, 1.0, outs=outs).item() for _ in range(3)}
    assert len(norms) == 1


def test_more_than_2_31_elements():
    g = torch.full(((1 << 31) + 5,), 0.5, dtype=torch.bfloat16, device="cuda")
    norm = clip_grad_norm([g], 1.0)
    n = 0.5 * ((1 << 31) + 5) ** 0.5
    assert abs(norm.item() - n) <= n * 2.0 ** -23
    want = torch.tensor(0.5 / (n + 1e-6), dtype=torch.float64)
    for at in (0, 1 << 30, (1 << 31) + 4):
        assert abs(g[at].double().cpu() - want) <= want * (2.0 ** -8 + 2.0 ** -22)


def test_captured_and_replayed():
    grads = make([70_000, 513, 20_000], DTYPES, seed=6)
    outs = [torch.empty_like(g, dtype=torch.float32) for g in grads]
    step = lambda: clip_grad_norm(grads, 2.0, outs=outs)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        for g, new in zip(grads, make([70_000, 513, 20_000], DTYPES, seed=20 + k)):
            g.copy_(new)
        eager = step().clone()
        want = [o.clone() for o in outs]
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, eager) and all(torch.equal(o, w) for o, w in zip(outs, want))


def test_with_a_process_group_of_one(tmp_path):
    import torch.distributed as dist
    if dist.is_initialized():
        pytest.skip("a process group exists already")
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/rendezvous", rank=0, world_size=1)
    try:
        grads = make([1000, 33], [torch.bfloat16])
        keep = [g.clone() for g in grads]
        assert grad_norm(grads, group=dist.group.WORLD).item() == grad_norm(grads).item()
        check(keep, grads, clip_grad_norm(grads, 1.0, group=dist.group.WORLD), 1.0)
    finally:
        dist.destroy_process_group()


def test_refusals():
    from transformer_engine_amd import NVTEError
    g = torch.ones(100, device="cuda")
    with pytest.raises(RuntimeError):
        grad_norm([g.cpu()])
    with pytest.raises(TypeError):
        grad_norm([g.double()])
    with pytest.raises(ValueError):
        grad_norm([torch.ones(10, 10, device="cuda").t()])
    with pytest.raises(ValueError):
        clip_grad_norm([g], 1.0, outs=[])
    with pytest.raises(ValueError):
        clip_grad_norm([g], 1.0, outs=[g[:50]])
    for bad in (-1.0, float("nan")):
        with pytest.raises(NVTEError, match="max_norm"):
            clip_grad_norm([g], bad)
    with pytest.raises(NVTEError, match="eps"):
        clip_grad_norm([g], 1.0, eps=-1.0)
    with pytest.raises(NVTEError, match="overlaps"):
        clip_grad_norm([g, g], 1.0)
    with pytest.raises(NVTEError, match="overlaps"):
        clip_grad_norm([g[:50]], 1.0, outs=[g[25:75]])
    with pytest.raises(NVTEError, match="dtype"):
        clip_grad_norm([g[:50]], 1.0, outs=[g.view(torch.bfloat16)[:50]])
    assert (g == 1).all()

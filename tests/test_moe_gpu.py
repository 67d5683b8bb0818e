"""A mixture-of-experts layer for a few tokens against the formulas in 64 bits.

Bounds are derived: a sum of n fp32 products is off by at most n 2^-23 times the sum of their magnitudes; |silu'| <= 1.1; the
sigmoid through 2^x and 1/x is off by 2^-20 + |g| 2^-23 of itself; h's two bf16 terms by 2^-16 of it; the result by half a step."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from transformer_engine_amd.moe import moe_forward, moe_topk


def make(t, h, f, e, k, dtype, fp8=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = randn(t, h).to(dtype)
    w1, w2 = randn(e, 2 * f, h) * h ** -0.5, randn(e, h, f) * f ** -0.5
    s1 = s2 = None
    if fp8:
        s1, s2 = (w.abs().amax(dim=(1, 2)) / 448 for w in (w1, w2))
        w1, w2 = (w / s[:, None, None] for w, s in ((w1, s1), (w2, s2)))
    wt = torch.float8_e4m3fn if fp8 else dtype
    ids = torch.stack([torch.randperm(e, generator=g, device="cuda")[:k] for _ in range(t)]).to(torch.int32) if t else \
        torch.empty(0, k, dtype=torch.int32, device="cuda")
    weights = torch.rand(t, k, generator=g, device="cuda")
    return x, w1.to(wt), w2.to(wt), ids, weights, s1, s2


def oracle(x, w1, w2, ids, weights, s1, s2):
    x = x.double()
    t, h = x.shape
    e, f2, _ = w1.shape
    f = f2 // 2
    out, mag = torch.zeros_like(x), torch.zeros_like(x)
    for i in range(e):
        row, col = (ids == i).nonzero(as_tuple=True)
        if row.numel() == 0:
            continue
        a, b = w1[i].double(), w2[i].double()
        if s1 is not None:
            a, b = a * s1[i].double(), b * s2[i].double()
        xr, wt = x[row], weights[row, col].double()[:, None]
        g, u = xr @ a[:f].t(), xr @ a[f:].t()
        dg, du = ((xr.abs() @ m.abs().t()) * (h + 2) * 2.0 ** -23 for m in (a[:f], a[f:]))
        z = g * torch.sigmoid(g) * u
        dz = 1.1 * dg * (u.abs() + du) + (g * torch.sigmoid(g)).abs() * du + z.abs() * (2.0 ** -16 + 2.0 ** -20 + g.abs() * 2.0 ** -23)
        out.index_add_(0, row, wt * (z @ b.t()))
        mag.index_add_(0, row, wt.abs() * (dz @ b.abs().t() + ((z.abs() + dz) @ b.abs().t()) * (f + 2 + ids.shape[1]) * 2.0 ** -23))
    return out, mag


def check(got, args):
    val, off = oracle(*args)
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * (val.abs() + off) + off + info.smallest_normal * info.eps
    err = (got.double() - val).abs()
    assert got.shape == val.shape
    assert (err <= bound).all(), f"{(err / bound.clamp(min=1e-300)).max().item():.3g} times its bound"


SHAPES = [  # tokens, hidden, ffn, experts, top_k
    (1, 64, 64, 1, 1),
    (1, 4096, 1024, 8, 2),
    (2, 16, 16, 4, 4),
    (3, 33, 17, 5, 2),
    (5, 2048, 704, 64, 8),
    (16, 520, 264, 8, 2),
    (17, 136, 1000, 3, 3),
    (33, 264, 520, 4, 1),
    (64, 512, 512, 8, 2),
    (70, 72, 40, 2, 2),
    (256, 64, 96, 16, 4),
    (256, 48, 80, 300, 16),
]


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp8", "fp8 fp16"])
@pytest.mark.parametrize("t,h,f,e,k", SHAPES)
def test_forward(t, h, f, e, k, kind):
    dtype = torch.float16 if "fp16" in kind else torch.bfloat16
    args = make(t, h, f, e, k, dtype, fp8="fp8" in kind, seed=t + h)
    x, w1, w2, ids, weights, s1, s2 = args
    check(moe_forward(x, w1, w2, ids, weights, s1, s2), args)


def test_raw_bytes_and_grouped_tensors_are_the_same_weights():
    from transformer_engine_amd.grouped import GroupedTensor, group_quantize
    from transformer_engine_amd.tensor import DType, Float8CurrentScalingQuantizer
    x, w1, w2, ids, weights, s1, s2 = make(6, 128, 64, 4, 2, torch.bfloat16, fp8=True)
    want = moe_forward(x, w1, w2, ids, weights, s1, s2)
    assert torch.equal(moe_forward(x, w1.view(torch.uint8), w2.view(torch.uint8), ids, weights, s1, s2), want)
    group = lambda w, s: GroupedTensor(num_tensors=4, logical_shape=(w.shape[0] * w.shape[1], w.shape[2]), dtype=torch.bfloat16,
                                       rowwise_data=w.view(torch.uint8).reshape(-1), scale_inv=s, fp8_dtype=DType.kFloat8E4M3)
    assert torch.equal(moe_forward(x, group(w1, s1), group(w2, s2), ids, weights), want)
    # what GroupedLinear's own weight quantizer makes
    hp = [torch.randn(4, *w.shape[1:], device="cuda", dtype=torch.bfloat16) * 0.1 for w in (w1, w2)]
    q = []
    for w in hp:
        quantizer = Float8CurrentScalingQuantizer(DType.kFloat8E4M3, torch.device("cuda"))
        quantizer.set_usage(rowwise=True, columnwise=False)
        q.append(group_quantize(w.view(-1, w.shape[2]), quantizer, 4))
    got = moe_forward(x, q[0], q[1], ids, weights)
    bytes_of = lambda g, w: g.rowwise_data.view(torch.float8_e4m3fn).view(w.shape)
    check(got, (x, bytes_of(q[0], w1), bytes_of(q[1], w2), ids, weights, q[0].scale_inv, q[1].scale_inv))


def test_ids_outside_the_experts_add_nothing_and_one_named_twice_counts_twice():
    x, w1, w2, ids, weights, _, _ = make(4, 64, 48, 4, 3, torch.bfloat16, seed=2)
    ids[0] = torch.tensor([-1, 2, 4], dtype=torch.int32)
    ids[1] = torch.tensor([3, 3, 1], dtype=torch.int32)
    ids[2] = torch.tensor([-1, 2 ** 31 - 1, 100], dtype=torch.int32)
    got = moe_forward(x, w1, w2, ids, weights)
    check(got, (x, w1, w2, ids, weights, None, None))
    assert (got[2] == 0).all()


def test_every_token_to_one_expert():
    x, w1, w2, ids, weights, _, _ = make(200, 64, 80, 3, 2, torch.bfloat16, seed=3)
    ids[:] = 1
    check(moe_forward(x, w1, w2, ids, weights), (x, w1, w2, ids, weights, None, None))


def test_non_finite_tokens_and_experts_stay_to_themselves():
    x, w1, w2, ids, weights, _, _ = make(20, 64, 80, 4, 2, torch.bfloat16, seed=4)
    ids[:, 0], ids[:, 1] = 0, 2
    ids[3] = torch.tensor([1, 3], dtype=torch.int32)
    want = moe_forward(x, w1, w2, ids, weights)
    x[3], w1[1], w2[3], x[7] = float("nan"), float("inf"), float("nan"), float("inf")
    got = moe_forward(x, w1, w2, ids, weights)
    good = torch.tensor([t for t in range(20) if t not in (3, 7)], device="cuda")
    assert torch.equal(got[good], want[good])
    assert not torch.isfinite(got[3].float()).any() and not torch.isfinite(got[7].float()).any()


def test_large_fp16_activations_pass_through():
    """silu(g) * u above fp16's largest number, brought back by a small second matrix."""
    x, w1, w2, ids, weights, _, _ = make(3, 64, 32, 2, 1, torch.float16, seed=5)
    w1, w2 = (w1.float() * 300).half(), (w2.float() * 2.0 ** -12).half()
    check(moe_forward(x, w1, w2, ids, weights), (x, w1, w2, ids, weights, None, None))
    z = x.float() @ w1[ids[0, 0]].float().t()
    assert (z[:, :32].abs() * z[:, 32:].abs()).max() > 65504


def test_leading_dims_strides_and_no_tokens():
    x, w1, w2, ids, weights, _, _ = make(6, 64, 48, 4, 2, torch.bfloat16, seed=6)
    want = moe_forward(x, w1, w2, ids, weights)
    wide = torch.zeros(2, 3, 80, dtype=x.dtype, device="cuda")
    wide[..., 8:72] = x.view(2, 3, 64)
    ids_t = ids.t().contiguous().t()
    assert torch.equal(moe_forward(wide[..., 8:72], w1, w2, ids_t, weights).view(6, 64), want)
    off = torch.cat([w1.new_zeros(1), w1.reshape(-1)])[1:].view(w1.shape)       # weights that are not 16-byte aligned
    check(moe_forward(x, off, w2, ids, weights), (x, w1, w2, ids, weights, None, None))
    assert moe_forward(x[:0], w1, w2, ids[:0], weights[:0]).shape == (0, 64)


def test_captured_and_replayed_with_new_routing():
    x, w1, w2, _, _, s1, s2 = make(12, 256, 128, 8, 2, torch.bfloat16, fp8=True, seed=7)
    logits = torch.randn(12, 8, device="cuda")
    def step():
        ids, weights = moe_topk(logits, 2)
        return ids, weights, moe_forward(x, w1, w2, ids, weights, s1, s2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        logits.copy_(torch.randn(12, 8, device="cuda"))
        x.copy_(torch.randn(12, 256, device="cuda"))
        eager = [v.clone() for v in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager))


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (3, 8, 2), (5, 64, 8), (7, 65, 5), (1000, 128, 4), (4, 256, 64), (9, 1000, 10), (2, 1024, 64)])
def test_topk(t, e, k, dtype, renormalize):
    g = torch.Generator(device="cuda").manual_seed(t + e)
    logits = (torch.randn(t, e, generator=g, device="cuda") * 3).to(dtype)      # 16-bit logits tie often
    ids, weights = moe_topk(logits, k, renormalize)
    want = logits.double().sort(dim=-1, descending=True, stable=True).indices[:, :k]
    assert ids.dtype == torch.int32 and torch.equal(ids.long(), want)
    p = torch.softmax(logits.double(), -1).gather(1, want)
    p = p / p.sum(-1, keepdim=True) if renormalize else p
    # exp is off by an ulp or two (2^-22) and by half a step of its argument (|x| 2^-24), the sum by e 2^-24, the quotient by 2^-24
    assert ((weights.double() - p).abs() <= p * (2.0 ** -21 + e * 2.0 ** -23 + 64 * 2.0 ** -23)).all()


def test_topk_of_equal_masked_and_bad_logits():
    inf, nan = float("inf"), float("nan")
    rows = [[0.0, -0.0, 0.0, 0.0], [-inf, 1.0, -inf, -inf], [nan, 1.0, 2.0, 3.0], [-inf] * 4, [nan] * 4]
    ids, weights = moe_topk(torch.tensor(rows, device="cuda"), 3)
    assert ids.tolist()[:3] == [[0, 1, 2], [1, 0, 2], [3, 2, 1]] and ids.tolist()[4] == [0, 1, 2]
    assert ids.tolist()[3] == [0, 1, 2]
    assert torch.allclose(weights[0], torch.full((3,), 1 / 3, device="cuda"))
    assert weights[1].tolist() == [1.0, 0.0, 0.0]
    assert weights[3].isnan().all() and weights[4].isnan().all()


def test_refusals():
    from transformer_engine_amd import NVTEError
    x, w1, w2, ids, weights, _, _ = make(4, 64, 48, 4, 2, torch.bfloat16)
    for bad, error in (
            ((x.float(), w1, w2, ids, weights), TypeError),
            ((x, w1.half(), w2, ids, weights), TypeError),
            ((x, w1[:, :95], w2, ids, weights), ValueError),
            ((x, w1, w2[:, :, :40], ids, weights), ValueError),
            ((x, w1, w2[:3], ids, weights), ValueError),
            ((x[:, :32], w1, w2, ids, weights), ValueError),
            ((x, w1, w2, ids[:3], weights[:3]), ValueError),
            ((x, w1, w2, ids, weights[:, :1]), ValueError),
            ((x, w1, w2, ids.long(), weights), TypeError),
            ((x, w1, w2, ids, weights.double()), TypeError),
            ((x, w1, w2, ids, weights, torch.ones(4, device="cuda")), ValueError),
            ((x, w1.view(torch.uint8)[:, :, :64], w2.view(torch.uint8)[:, :, :48], ids, weights), ValueError),
            ((x, w1.transpose(1, 2).contiguous().transpose(1, 2), w2, ids, weights), ValueError),
            ((x.cpu(), w1, w2, ids, weights), (RuntimeError, ValueError))):
        with pytest.raises(error):
            moe_forward(*bad)
    big = make(257, 16, 16, 2, 1, torch.bfloat16)
    with pytest.raises(NVTEError, match="256"):
        moe_forward(*big[:5])
    with pytest.raises(ValueError, match="top_k"):
        moe_topk(torch.zeros(2, 4, device="cuda"), 5)
    with pytest.raises(NVTEError, match="1024"):
        moe_topk(torch.zeros(2, 1025, device="cuda"), 1)
    with pytest.raises(TypeError):
        moe_topk(torch.zeros(2, 4, device="cuda", dtype=torch.float64), 1)

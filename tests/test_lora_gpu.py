"""Low-rank adapters beside a shared projection against the formulas in 64 bits.

Bounds are derived, element by element: a sum of n fp32 products is off by at most n 2^-23 times the sum of their magnitudes
(2^-24 per operation, doubled for the matrix instruction's own order), a rank vector's two bf16 terms by 2^-16 of it (2^-17 each
for the split and, in fp16, for the term left out), and the result's one rounding by half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from transformer_engine_amd.lora import LoRALinear, lora, lora_backward, lora_forward


def make(t, k, o, r, n, dtype, seed=0, ids="mixed", std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda").mul_(std).to(dtype)
    x, base, dy, gbase = randn(t, k), randn(t, o), randn(t, o), randn(t, k)
    a, b = randn(n, r, k), randn(n, o, r)
    scaling = torch.rand(n, generator=g, device="cuda") + 0.25
    if ids == "mixed":
        i = torch.randint(-1, n, (t,), generator=g, device="cuda", dtype=torch.int32)
    elif ids == "runs":
        i = (torch.arange(t, device="cuda") * n // max(t, 1)).to(torch.int32)
    else:
        i = torch.full((t,), ids, device="cuda", dtype=torch.int32)
    return x, a, b, i, scaling, base, dy, gbase


def oracle(x, a, b, ids, scaling, base, dy, gbase):
    """(value, magnitude of the summed terms) of y, dx, da, db in 64 bits; dicts by name."""
    t, k = x.shape
    n, r, _ = a.shape
    o = b.shape[1]
    x, a, b, scaling, base, dy, gbase = (None if v is None else v.double() for v in (x, a, b, scaling, base, dy, gbase))
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=x.device)
    val = {"y": z(t, o) if base is None else base.clone(), "dx": z(t, k) if gbase is None else gbase.clone(),
           "da": z(n, r, k), "db": z(n, o, r)}
    mag = {key: torch.zeros_like(v) for key, v in val.items()}
    for i in range(n):
        rows = (ids == i).nonzero()[:, 0]
        if rows.numel() == 0:
            continue
        s = 1.0 if scaling is None else scaling[i]
        xi, dyi = x[rows], dy[rows]
        v, va = s * (xi @ a[i].t()), s * (xi.abs() @ a[i].abs().t())
        u, ua = s * (dyi @ b[i]), s * (dyi.abs() @ b[i].abs())
        val["y"][rows] += v @ b[i].t()
        mag["y"][rows] += va @ b[i].abs().t()
        val["dx"][rows] += u @ a[i]
        mag["dx"][rows] += ua @ a[i].abs()
        val["da"][i], mag["da"][i] = u.t() @ xi, ua.t() @ xi.abs()
        val["db"][i], mag["db"][i] = dyi.t() @ v, dyi.abs().t() @ va
    return val, mag


def check(name, got, val, mag, terms):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps   # a subnormal's step
    off = (2.0 ** -16 + terms * 2.0 ** -23) * mag
    bound = half * (val.abs() + off) + off + tiny + 2.0 ** -23 * val.abs()
    err = (got.double() - val).abs()
    assert got.shape == val.shape
    worst = (err / bound.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert (err <= bound).all(), f"{name}: {worst:.3g} times its bound"


def check_all(args, y, dx, da, db):
    x, a, b = args[0], args[1], args[2]
    t, k, (n, r, _), o = x.shape[0], x.shape[1], a.shape, b.shape[1]
    val, mag = oracle(*args)
    check("y", y, val["y"], mag["y"], k + r + 2)
    check("dx", dx, val["dx"], mag["dx"], o + r + 2)
    check("da", da, val["da"], mag["da"], o + t + 2)
    check("db", db, val["db"], mag["db"], k + t + 2)


SHAPES = [  # tokens, in, out, rank, adapters
    (1, 64, 64, 8, 1),
    (1, 4096, 512, 16, 8),
    (2, 1, 1, 1, 2),
    (15, 33, 7, 3, 4),
    (16, 256, 128, 16, 3),
    (17, 1000, 1032, 20, 5),
    (64, 136, 520, 64, 64),
    (65, 519, 130, 5, 2),
    (100, 72, 2056, 33, 7),
    (130, 648, 640, 128, 3),
    (333, 128, 136, 100, 2),
    (700, 2056, 264, 12, 40),
    (520, 96, 104, 4, 300),
    (1500, 520, 1100, 32, 6),
    (2100, 9, 1030, 128, 4),
    (1100, 7, 5, 66, 3),
    (4500, 264, 512, 24, 3),
    (4100, 136, 72, 64, 1),
    (4096, 40, 24, 8, 70),
    (8200, 24, 40, 8, 4096),
]


@pytest.mark.parametrize("ids", ["mixed", "runs"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k,o,r,n", SHAPES)
def test_forward_backward(t, k, o, r, n, dtype, ids):
    args = make(t, k, o, r, n, dtype, seed=t + k, ids=ids, std=0.5)
    x, a, b, i, scaling, base, dy, gbase = args
    y, saved = lora_forward(x, a, b, i, scaling, base=base)
    dx, da, db = lora_backward(dy, saved, base_grad=gbase)
    assert dx.dtype == da.dtype == db.dtype == dtype
    check_all(args, y, dx, da, db)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_no_base_no_scaling_fp32_gradients(dtype):
    x, a, b, i, _, _, dy, _ = make(77, 200, 312, 16, 4, dtype, seed=3)
    y, saved = lora_forward(x, a, b, i)
    dx, da, db = lora_backward(dy, saved, grad_dtype=torch.float32)
    assert da.dtype == db.dtype == torch.float32
    check_all((x, a, b, i, None, None, dy, None), y, dx, da, db)
    assert (y[i < 0] == 0).all() and (dx[i < 0] == 0).all()


@pytest.mark.parametrize("t", [50, 1300])
def test_rows_without_adapter_keep_the_base_bits(t):
    x, a, b, i, s, base, dy, gbase = make(t, 64, 96, 8, 2, torch.bfloat16, ids=-1)
    i[3], i[7], i[20] = 2, 2 ** 31 - 1, -2 ** 31        # all outside [0, 2)
    base[5, :50], gbase[6, 10:] = -0.0, -0.0
    y, saved = lora_forward(x, a, b, i, s, base=base)
    dx, da, db = lora_backward(dy, saved, base_grad=gbase)
    bits = lambda v: v.view(torch.int16)
    assert torch.equal(bits(y), bits(base)) and torch.equal(bits(dx), bits(gbase))
    assert (da == 0).all() and (db == 0).all()


@pytest.mark.parametrize("t", [40, 1000])
def test_adapters_without_tokens_get_zero_gradients_over_old_memory(t):
    x, a, b, i, s, base, dy, _ = make(t, 72, 80, 8, 6, torch.float16, ids=4)
    torch.full((6, 8, 72), float("nan"), dtype=torch.float16, device="cuda")   # freed at once: what the allocator may hand out
    y, saved = lora_forward(x, a, b, i, s, base=base)
    _, da, db = lora_backward(dy, saved)
    keep = torch.tensor([0, 1, 2, 3, 5], device="cuda")
    assert (da[keep] == 0).all() and (db[keep] == 0).all() and (da[4] != 0).any()


@pytest.mark.parametrize("t", [5, 40, 1100])
def test_non_finite_values_stay_in_their_rows(t):
    """Other requests' adapters and activations hold NaN and Inf: nobody else's results change by a bit."""
    args = make(t, 144, 272, 16, 4, torch.bfloat16, seed=9, ids="mixed")
    x, a, b, i, s, base, dy, gbase = args
    i[0], i[1] = 1, 2
    def run():
        y, saved = lora_forward(x, a, b, i, s, base=base)
        return (y, *lora_backward(dy, saved, base_grad=gbase))
    y0, dx0, da0, db0 = run()
    bad = i == 1
    x[bad] = float("nan")
    dy[bad] = float("inf")
    a[1] = float("inf")
    b[1] = float("nan")
    y1, dx1, da1, db1 = run()
    assert torch.equal(y0[~bad], y1[~bad]) and torch.equal(dx0[~bad], dx1[~bad])
    others = torch.tensor([0, 2, 3], device="cuda")
    assert torch.equal(da0[others], da1[others]) and torch.equal(db0[others], db1[others])
    assert not torch.isfinite(y1[bad].float()).any() and not torch.isfinite(dx1[bad].float()).any()


def test_small_fp16_gradients_do_not_vanish():
    """Rank vectors far below fp16's smallest number still reach gradients that fp32 holds."""
    args = make(64, 96, 128, 8, 2, torch.float16, seed=4)
    x, a, b, i, s, base, dy, gbase = args
    dy = (dy.float() * 2.0 ** -20).half()
    b = (b.float() * 2.0 ** -10).half()
    y, saved = lora_forward(x, a, b, i, s, base=base)
    dx, da, db = lora_backward(dy, saved, base_grad=None, grad_dtype=torch.float32)
    val, mag = oracle(x, a, b, i, s, base, dy, None)
    check("da", da, val["da"], mag["da"], 128 + 64 + 2)
    check("db", db, val["db"], mag["db"], 96 + 64 + 2)
    assert (da.abs().amax(dim=(1, 2)) > 0).all()


def test_large_fp16_rank_vectors_do_not_overflow():
    x, a, b, i, s, base, dy, gbase = make(20, 512, 64, 8, 1, torch.float16, seed=5, ids=0)
    x, b = x * 200, b * 2.0 ** -14
    a = a.abs() * 16
    x = x.abs()
    y, _ = lora_forward(x, a, b, i, s, base=base)
    val, mag = oracle(x, a, b, i, s, base, dy, gbase)
    assert (x[:1].float() @ a[0, :1].float().t()).item() > 65504
    check("y", y, val["y"], mag["y"], 512 + 8 + 2)


def test_strided_inputs_leading_dims_and_in_place_output():
    x, a, b, i, s, base, dy, gbase = make(24, 64, 96, 8, 3, torch.bfloat16, seed=6)
    ref, saved = lora_forward(x, a, b, i, s, base=base)
    ref_grads = lora_backward(dy, saved, base_grad=gbase)
    wide = torch.zeros(4, 6, 128, dtype=x.dtype, device="cuda")
    wide[..., 32:96] = x.view(4, 6, 64)
    at = a.transpose(1, 2).contiguous().transpose(1, 2)
    y, saved = lora_forward(wide[..., 32:96], at, b, i.view(4, 6), s, base=base.view(4, 6, 96))
    assert torch.equal(y.view(24, 96), ref)
    grads = lora_backward(dy.view(4, 6, 96), saved, base_grad=gbase.view(4, 6, 64))
    for g, r in zip(grads, ref_grads):
        assert torch.equal(g.reshape(r.shape), r)
    buf = base.clone()
    y, saved = lora_forward(x, a, b, i, s, base=buf, out=buf, needs_backward=False)
    assert y is buf and saved is None and torch.equal(buf, ref)


@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("o", [96, 1029, 2052])
def test_in_place_of_a_large_batch(o, n):
    x, a, b, i, s, base, _, _ = make(1400, 64, o, 8, n, torch.bfloat16, seed=17)
    ref, _ = lora_forward(x, a, b, i, s, base=base)
    buf = base.clone()
    lora_forward(x, a, b, i, s, base=buf, out=buf)
    assert torch.equal(buf, ref)
    none, _ = lora_forward(x, a, b, i, s)
    zero, _ = lora_forward(x, a, b, i, s, base=torch.zeros_like(base))
    assert torch.equal(none, zero) and (none[i < 0] == 0).all()


def test_the_order_of_the_tokens_does_not_change_a_row():
    """A large mixed batch, its tokens put in another order: the same rows, and gradients within their bounds."""
    args = make(3000, 264, 392, 16, 20, torch.bfloat16, seed=18)
    x, a, b, i, s, base, dy, gbase = args
    p = torch.randperm(3000, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    y0, saved = lora_forward(x, a, b, i, s, base=base)
    dx0, _, _ = lora_backward(dy, saved, base_grad=gbase)
    y1, saved = lora_forward(x[p], a, b, i[p], s, base=base[p])
    dx1, da1, db1 = lora_backward(dy[p], saved, base_grad=gbase[p])
    assert torch.equal(y0[p], y1) and torch.equal(dx0[p], dx1)
    check_all(args, y0, dx0, da1, db1)


@pytest.mark.parametrize("off", [1, 4])
def test_misaligned_storage(off):
    """Every operand starts `off` elements into its storage."""
    args = make(37, 88, 104, 16, 3, torch.bfloat16, seed=8)
    x, a, b, i, s, base, dy, gbase = args
    shift = lambda v: torch.cat([v.new_zeros(off), v.reshape(-1)])[off:].view(v.shape)
    y, saved = lora_forward(shift(x), shift(a), shift(b), i, s, base=shift(base))
    dx, da, db = lora_backward(shift(dy), saved, base_grad=shift(gbase))
    check_all(args, y, dx, da, db)
    buf = shift(base)
    out, _ = lora_forward(x, a, b, i, s, base=buf, out=buf)
    assert torch.equal(out, y)


def test_no_tokens():
    x, a, b, i, s, base, dy, gbase = make(0, 64, 96, 8, 3, torch.bfloat16)
    y, saved = lora_forward(x, a, b, i, s, base=base)
    dx, da, db = lora_backward(dy, saved, base_grad=gbase)
    assert y.shape == (0, 96) and dx.shape == (0, 64) and (da == 0).all() and (db == 0).all()


def test_only_one_direction_is_asked_for():
    x, a, b, i, s, base, dy, gbase = make(30, 64, 96, 8, 3, torch.bfloat16)
    _, saved = lora_forward(x, a, b, i, s, base=base)
    dx, da, db = lora_backward(dy, saved, base_grad=gbase)
    assert lora_backward(dy, saved, requires_dgrad=False)[0] is None
    assert torch.equal(lora_backward(dy, saved, requires_dgrad=False)[1], da)
    only = lora_backward(dy, saved, base_grad=gbase, requires_wgrad=False)
    assert only[1] is None and only[2] is None and torch.equal(only[0], dx)


def test_the_same_call_gives_the_same_bits():
    args = make(3000, 520, 640, 16, 9, torch.bfloat16, seed=11)
    x, a, b, i, s, base, dy, gbase = args
    runs = []
    for _ in range(3):
        y, saved = lora_forward(x, a, b, i, s, base=base)
        runs.append((y, *lora_backward(dy, saved, base_grad=gbase)))
    for other in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(runs[0], other))


def test_offsets_beyond_32_bits():
    t, k, o, r = 150_001, 16, 14336, 4                       # base and y hold 2.15e9 elements
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(t, k, generator=g, device="cuda").to(torch.bfloat16)
    a = torch.randn(2, r, k, generator=g, device="cuda").to(torch.bfloat16)
    b = torch.randn(2, o, r, generator=g, device="cuda").to(torch.bfloat16)
    i = (torch.arange(t, device="cuda") % 2).to(torch.int32)
    base = torch.ones(t, o, dtype=torch.bfloat16, device="cuda")
    y, saved = lora_forward(x, a, b, i, base=base, out=base)
    rows = torch.tensor([0, 1, t // 2, t - 2, t - 1], device="cuda")
    val, mag = oracle(x[rows], a, b, i[rows], None, torch.ones(5, o, dtype=torch.bfloat16, device="cuda"), y[rows], None)
    check("y", y[rows], val["y"], mag["y"], k + r + 2)
    dx, _, _ = lora_backward(y, saved, requires_wgrad=False)
    val, mag = oracle(x[rows], a, b, i[rows], None, None, y[rows], None)
    check("dx", dx[rows], val["dx"], mag["dx"], o + r + 2)


def test_gradients_against_differences():
    """d/de of sum(y * dy) along random directions, from forward passes alone (fp16, small values, 2nd-order central differences)."""
    x, a, b, i, s, base, dy, _ = make(32, 64, 48, 8, 2, torch.float16, seed=12)
    _, saved = lora_forward(x, a, b, i, s)
    dx, da, db = lora_backward(dy, saved, grad_dtype=torch.float32)
    def f(x, a, b):   # the same formula in 64 bits: the kernel's forward is checked against it above
        val, _ = oracle(x, a, b, i, s, None, dy, None)
        return (val["y"] * dy.double()).sum()
    g = torch.Generator(device="cuda").manual_seed(2)
    for grad, which in ((dx, 0), (da, 1), (db, 2)):
        args = [x.double(), a.double(), b.double()]
        d = torch.randn(args[which].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-4
        plus, minus = list(args), list(args)
        plus[which], minus[which] = args[which] + h * d, args[which] - h * d
        num = (f(*plus) - f(*minus)) / (2 * h)
        ana = (grad.double() * d).sum()
        # every entry of grad is off by at most 2^-11 of itself (fp16) and 2^-12 of its terms; f is linear in each argument
        assert abs(num - ana) <= 2.0 ** -10 * (grad.double().abs() * d.abs()).sum() + 1e-6 * abs(num)


def test_autograd_matches_the_bare_passes():
    x, a, b, i, s, base, dy, _ = make(45, 64, 96, 8, 3, torch.bfloat16, seed=13)
    xs = [v.clone().requires_grad_() for v in (x, a, b, base)]
    y = lora(xs[0], xs[1], xs[2], i, s, xs[3])
    y.backward(dy)
    y0, saved = lora_forward(x, a, b, i, s, base=base)
    dx, da, db = lora_backward(dy, saved)
    assert torch.equal(y, y0)
    for v, g in zip(xs, (dx, da, db, dy)):
        assert torch.equal(v.grad, g)
    y = lora(x, xs[1], b, i, s, base)
    xs[1].grad = None
    y.backward(dy.t().contiguous().t())                      # another memory order
    assert torch.equal(xs[1].grad, da)


@pytest.mark.parametrize("t", [1, 300, 1300])
def test_captured_and_replayed(t):
    x, a, b, i, s, base, dy, gbase = make(t, 264, 392, 16, 5, torch.bfloat16, seed=14)
    def step():
        y, saved = lora_forward(x, a, b, i, s, base=base)
        return (y, *lora_backward(dy, saved, base_grad=gbase))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    g = torch.Generator(device="cuda").manual_seed(15)
    for _ in range(4):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        i.copy_(torch.randint(-1, 5, i.shape, generator=g, device="cuda"))
        eager = [v.clone() for v in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager))


def test_runs_on_the_callers_stream():
    args = make(600, 520, 640, 16, 5, torch.bfloat16, seed=16)
    x, a, b, i, s, base, dy, gbase = args
    want, saved = lora_forward(x, a, b, i, s, base=base)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        late = torch.zeros_like(x)
        torch.cuda._sleep(2_000_000)
        late.copy_(x)
        got, _ = lora_forward(late, a, b, i, s, base=base)
    stream.synchronize()
    assert torch.equal(got, want)


def test_module_beside_a_frozen_linear():
    torch.manual_seed(0)
    m = LoRALinear(256, 384, rank=8, num_adapters=3, alpha=16.0)
    x = torch.randn(64, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ids = torch.randint(-1, 3, (64,), device="cuda", dtype=torch.int32)
    assert [n for n, p in m.named_parameters() if p.requires_grad] == ["lora_a", "lora_b"]
    assert torch.allclose(m.scaling, torch.full((3,), 2.0, device="cuda"))
    y0 = m(x, ids)
    with torch.no_grad():
        torch.nn.init.normal_(m.lora_b, std=0.2)
    from transformer_engine_amd.linear import linear_backward, linear_forward
    from transformer_engine_amd.tensor import Float8Quantizer  # noqa: F401  (the recipe's quantizers)
    y = m(x, ids)
    dy = torch.randn_like(y)
    y.backward(dy)
    assert m.linear.weight.grad is None and x.grad is not None
    # the adapters' part on top of the shared projection, both within FP8's own error of the unquantized formula
    w = m.linear.weight.double()
    val, mag = oracle(x.detach(), m.lora_a.detach(), m.lora_b.detach(), ids, m.scaling,
                      (x.detach().double() @ w.t()), dy, dy.double() @ w)
    rel = lambda got, want: ((got.double() - want).norm() / want.norm()).item()
    assert rel(y, val["y"]) < 2.0 ** -4 and rel(x.grad, val["dx"]) < 2.0 ** -3   # half a step of e4m3, of e5m2
    check("da", m.lora_a.grad, val["da"], mag["da"], 384 + 64 + 2)
    check("db", m.lora_b.grad, val["db"], mag["db"], 256 + 64 + 2)
    assert torch.isfinite(y0.float()).all()


def _gpu_args():
    return make(8, 64, 96, 8, 3, torch.bfloat16)


@pytest.mark.parametrize("change, error", [
    (dict(x=lambda v: v.float()), TypeError),
    (dict(a=lambda v: v.half()), TypeError),
    (dict(a=lambda v: v[:, :, :32]), ValueError),
    (dict(b=lambda v: v[:2]), ValueError),
    (dict(ids=lambda v: v.long()), TypeError),
    (dict(ids=lambda v: v[:4]), ValueError),
    (dict(s=lambda v: v.double()), ValueError),
    (dict(s=lambda v: v[:2]), ValueError),
    (dict(base=lambda v: v[:, :64]), ValueError),
    (dict(base=lambda v: v.float()), TypeError),
    (dict(x=lambda v: v.cpu()), (RuntimeError, ValueError)),
])
def test_refusals(change, error):
    x, a, b, i, s, base, _, _ = _gpu_args()
    args = dict(x=x, a=a, b=b, ids=i, s=s, base=base)
    for name, f in change.items():
        args[name] = f(args[name])
    with pytest.raises(error):
        lora_forward(args["x"], args["a"], args["b"], args["ids"], args["s"], base=args["base"])


def test_refuses_an_output_over_an_input():
    buf = torch.zeros(8 * 64 + 32, dtype=torch.bfloat16, device="cuda")
    x, a, b, i, s, _, _, _ = make(8, 64, 64, 8, 3, torch.bfloat16)
    with pytest.raises(ValueError, match="overlaps x"):
        lora_forward(x, a, b, i, s, out=x)
    with pytest.raises(ValueError, match="overlaps base"):
        lora_forward(x, a, b, i, s, base=buf[:512].view(8, 64), out=buf[32:].view(8, 64))


def test_refuses_large_ranks_and_too_many_trained_adapters():
    from transformer_engine_amd import NVTEError
    x, a, b, i, s, _, dy, _ = make(4, 16, 16, 129, 1, torch.bfloat16)
    with pytest.raises(NVTEError, match="rank"):
        lora_forward(x, a, b, i, s)
    x, a, b, i, s, _, dy, _ = make(4, 8, 8, 1, 4097, torch.bfloat16)
    _, saved = lora_forward(x, a, b, i, s)
    with pytest.raises(NVTEError, match="4096"):
        lora_backward(dy, saved)
    assert lora_backward(dy, saved, requires_wgrad=False)[0] is not None

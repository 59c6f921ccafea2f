"""Dense operators on the GPU against their 64-bit values (tests/dense_oracle.py has the tolerances)."""
import ctypes as C

import pytest
import torch

import dartmoq_b200 as D
import dense_oracle as R
from dartmoq_b200 import _lib, dense, synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = (torch.bfloat16, torch.float16)


def rng(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def acts(g, t, k, dtype):
    x = torch.randn(t, k, generator=g)
    x[:, torch.rand(k, generator=g) < 0.01] *= 20
    return x.to(dtype).to(DEV)


def weight8(g, n, k):
    codes = (torch.randn(n, k, generator=g) * 32).round().clamp(-127, 127).to(torch.int8)
    return codes.to(DEV), (0.02 / 32 * torch.exp(0.3 * torch.randn(n, generator=g))).to(DEV)


def healthy():
    D.WxA16BitPartitionedGroupMoE.check_device_status()


# --------------------------------------------------------------------------------------------- quantiser

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,k", [(1, 16), (3, 128), (77, 2064), (5, 8192), (2, 40000)])
def test_quantize_codes_equal_the_definition(t, k, dtype):
    x = acts(rng(t * k), t, k, dtype)
    codes, scale = dense.quantize_int8_tokens(x)
    want, s = R.quantize(x)
    assert codes.dtype == torch.int8 and scale.dtype == torch.float32 and scale.shape == (t,)
    assert torch.equal(codes.double().cpu(), want)
    assert torch.equal(scale.cpu(), s.float())                     # max / 127, correctly rounded


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_special_rows(dtype):
    fi = torch.finfo(dtype)
    k = 256
    x = torch.zeros(9, k)
    x[1] = torch.arange(k) * 0.5 - 64.0                            # with max 127 every odd entry is a tie
    x[1, 0] = 127.0
    x[2], x[2, 3] = fi.max / 3, -fi.max
    x[3], x[3, 5] = fi.smallest_normal, fi.smallest_normal * fi.eps * 3   # subnormals
    x[4] = fi.smallest_normal * fi.eps                             # the smallest number everywhere
    x[5, 7] = float("nan")
    x[6, k - 1] = float("-inf")
    x[7, 100] = 1.0
    x[8] = torch.randn(k, generator=rng(1)) * 1e-3
    x = x.to(dtype).to(DEV)
    codes, scale = dense.quantize_int8_tokens(x)
    fine = [0, 1, 2, 3, 4, 7, 8]
    want, s = R.quantize(x[fine])
    assert torch.equal(codes[fine].double().cpu(), want) and torch.equal(scale[fine].cpu(), s.float())
    assert int(codes[[0, 5, 6]].abs().max()) == 0 and torch.isnan(scale[[5, 6]]).all() and float(scale[0]) == 0.0
    w, ws = weight8(rng(2), 24, k)
    y = dense.int8_linear(x, w, ws)
    assert torch.isnan(y[[5, 6]]).all() and torch.isfinite(y[[0, 1, 4, 7, 8]]).all() and float(y[0].abs().max()) == 0.0


def test_quantize_shapes_and_strides():
    g = rng(3)
    big = randn(g, 6, 5, 320, dtype=torch.bfloat16)
    codes, scale = dense.quantize_int8_tokens(big[:, 1:4, :128])    # rows that do not follow one another
    want, s = R.quantize(big[:, 1:4, :128])
    assert codes.shape == (6, 3, 128) and scale.shape == (6, 3)
    assert torch.equal(codes.double().cpu(), want) and torch.equal(scale.cpu(), s.float())
    for view in (big[:, 0, 8:136], big[:, 0, 3:131], big[0, :, :64].t()[:, :1].expand(64, 16), big[:, :, 5:21].transpose(0, 1)):
        codes, scale = dense.quantize_int8_tokens(view)
        assert torch.equal(codes.double().cpu(), R.quantize(view)[0])
    vec, s = dense.quantize_int8_tokens(big[0, 0])
    assert vec.shape == (320,) and s.shape == ()
    none, s = dense.quantize_int8_tokens(big[:0])
    assert none.shape == (0, 5, 320) and s.shape == (0, 5)


# --------------------------------------------------------------------------------------------- 8-bit products

SIZES8 = [(1, 1, 16), (1, 33, 128), (2, 512, 2048), (7, 1001, 144), (16, 256, 2064), (17, 96, 4096), (32, 100, 1040), (64, 640, 512), (65, 257, 3600), (127, 130, 272),
          (129, 257, 1024), (300, 1001, 2064), (700, 4096, 256), (1300, 2200, 640), (1545, 2201, 144), (9, 40, 1040),
          (3, 24, 5200), (16, 33, 9104), (8, 70, 1024), (12, 9000, 2048),
          (130, 1000, 528), (256, 333, 2064)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", (False, True))
@pytest.mark.parametrize("t,n,k", SIZES8)
def test_int8_linear(t, n, k, bias, dtype):
    g = rng(t + n + k)
    x, (w, ws) = acts(g, t, k, dtype), weight8(g, n, k)
    b = randn(g, n, dtype=dtype) if bias else None
    y = dense.int8_linear(x, w, ws, b)
    codes, s = R.quantize(x)
    prod = (codes @ w.double().cpu().t()) * s[:, None] * ws.double().cpu()
    want = prod + (b.double().cpu() if bias else 0)
    # one rounding to 16 bits of a value that carries five 32-bit roundings (sum to float, two scales, scale / 127, bias);
    # smallest_normal * eps is a step below the normal numbers
    fi = torch.finfo(dtype)
    e32 = 5 * 2.0 ** -24 * (prod.abs() + want.abs())
    tol = fi.eps / 2 * (want.abs() + e32) + e32 + fi.smallest_normal * fi.eps
    assert y.shape == (t, n) and y.dtype == dtype
    assert ((y.double().cpu() - want).abs() <= tol).all()
    q, sc = dense.quantize_int8_tokens(x)
    assert torch.equal(dense.int8_matmul(q, sc, w, ws, b, out_dtype=dtype), y)
    healthy()


def test_int8_sums_are_exact_at_the_largest_inner_size():
    k = 131056
    codes = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((20, k), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    w[2, ::2] = 127
    one = torch.ones(20, device=DEV)
    y = dense.int8_matmul(codes, torch.full((3,), 2.0 ** -20, device=DEV), w, one, out_dtype=torch.bfloat16)
    want = (codes.double() @ w.double().t()).cpu() * 2.0 ** -20
    assert ((y.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() * (1 + 2.0 ** -22)).all()
    with pytest.raises(_lib.DmoqError):
        wide = torch.zeros((1, k + 16), dtype=torch.int8, device=DEV)
        dense.int8_matmul(wide, torch.ones(1, device=DEV), wide, one[:1])


def test_inner_sizes_past_32_bits_are_refused():
    """2^32 + 16 columns are not 16 (the tensors hold one element each)."""
    k = (1 << 32) + 16
    x = torch.ones(1, dtype=torch.bfloat16, device=DEV).expand(1, k)
    w, one = torch.ones(1, dtype=torch.int8, device=DEV).expand(1, k), torch.ones(1, device=DEV)
    for call in (lambda: dense.quantize_int8_tokens(x), lambda: dense.int8_linear(x, w, one), lambda: dense.int8_matmul(w, one, w, one),
                 lambda: dense.int8_gated_linear(x, w, one, w, one)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("t", (1, 12, 40, 200, 2500))
def test_int8_scales_whose_product_leaves_the_32_bit_range(t):
    """Token and row scales far apart: their product alone underflows or overflows, the result does not."""
    g = rng(90 + t)
    n, k = 300, 528
    codes = torch.randint(-127, 128, (t, k), generator=g).to(torch.int8).to(DEV)
    w = torch.randint(-127, 128, (n, k), generator=g).to(torch.int8).to(DEV)
    w[5] = 0                                                        # sums of zero
    scale = torch.tensor([7.9e-33, 2.0 ** -61, 2e36, 1.0, 0.0, 3e-41, 1e20])[torch.arange(t) % 7].to(DEV)
    row = torch.tensor([1e-12, 1e3, 2.0 ** 48, 0.01, 1e-38, 3e24, 2.0 ** -75, 0.0])[torch.arange(n) % 8].to(DEV)
    y = dense.int8_matmul(codes, scale, w, row)
    sums = codes.double() @ w.double().t()
    want = (sums * scale.double()[:, None] * row.double()).cpu()
    got, fi = y.double().cpu(), torch.finfo(torch.bfloat16)
    finite = want.abs() < fi.max + 2.0 ** 119                       # half a step beyond the largest number rounds to it
    # one rounding to 16 bits, four to 32 (the sum, two products, the result); below the normal numbers a step is not relative
    tol = want.abs() * (2.0 ** -8 + 4 * 2.0 ** -24) + fi.smallest_normal * fi.eps
    assert ((got - want).abs() <= tol)[finite].all()
    assert torch.equal(got[~finite], torch.sign(want[~finite]) * float("inf"))
    assert torch.equal(y[:, 3::8][3::7], dense.int8_matmul(codes[3::7], scale[3::7], w[3::8], row[3::8]))   # whatever the neighbours are
    # gates: tokens 2^-100 times as large and row scales 2^100 times as large leave the 64-bit values as they are
    x, (wg, sg), (wu, su) = acts(g, t, k, torch.bfloat16), weight8(g, n, k), weight8(g, n, k)
    h = dense.int8_gated_linear(x * 2.0 ** -100, wg, sg * 2.0 ** 100, wu, su * 2.0 ** 100)
    q, s = R.quantize(x)
    gate, up = ((q @ m.double().cpu().t()) * s[:, None] * sm.double().cpu() for m, sm in ((wg, sg), (wu, su)))
    want = R.silu(gate) * up
    e32 = 2.0 ** -24 * (4 * (1 + gate.abs()) + 4 + 2 * (2 + gate.abs()) + 5)     # as for int8_gated_linear
    assert ((h.double().cpu() - want).abs() <= want.abs() * (2.0 ** -8 * (1 + e32) + e32) + fi.smallest_normal * fi.eps).all()
    healthy()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", SIZES8)
def test_int8_gated_linear(t, n, k, dtype):
    g = rng(t * n + k)
    x, (wg, sg), (wu, su) = acts(g, t, k, dtype), weight8(g, n, k), weight8(g, n, k)
    sg, su = sg * (64 / k) ** 0.5 * 4, su * (64 / k) ** 0.5         # gates of a few units at every inner size
    h = dense.int8_gated_linear(x, wg, sg, wu, su)
    codes, s = R.quantize(x)
    gate = (codes @ wg.double().cpu().t()) * s[:, None] * sg.double().cpu()
    up = (codes @ wu.double().cpu().t()) * s[:, None] * su.double().cpu()
    want = R.silu(gate) * up
    # silu's relative condition is at most 1 + |g|; g carries four 32-bit roundings, u four, the exponential 2 + |g| and the
    # quotient and products five
    fi = torch.finfo(dtype)
    e32 = 2.0 ** -24 * (4 * (1 + gate.abs()) + 4 + 2 * (2 + gate.abs()) + 5)
    tol = want.abs() * (fi.eps / 2 * (1 + e32) + e32) + fi.smallest_normal * fi.eps
    assert h.shape == (t, n) and ((h.double().cpu() - want).abs() <= tol).all()
    healthy()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,n,k", SIZES8)
def test_int8_gated_matmul(t, n, k, dtype):
    """Of the tokens' own codes: bit for bit what the quantiser in front of the same products gives."""
    g = rng(t * n + k + 1)
    x, (wg, sg), (wu, su) = acts(g, t, k, dtype), weight8(g, n, k), weight8(g, n, k)
    codes, scale = dense.quantize_int8_tokens(x)
    h = dense.int8_gated_matmul(codes, scale, wg, sg, wu, su, out_dtype=dtype)
    assert h.shape == (t, n) and h.dtype == dtype
    assert torch.equal(h, dense.int8_gated_linear(x, wg, sg, wu, su))
    healthy()


def test_int8_gated_matmul_shapes_strides_and_refusals():
    g = rng(63)
    codes = torch.randint(-128, 128, (4, 6, 512), generator=g).to(torch.int8).to(DEV)
    scale = (torch.rand(4, 6, generator=g) * 1e-3).to(DEV)
    (wg, sg), (wu, su) = weight8(g, 57, 512), weight8(g, 57, 512)
    want = dense.int8_gated_matmul(codes[:, ::2, 16:272].contiguous(), scale[:, ::2].contiguous(), wg[:, :256].contiguous(), sg,
                                   wu[:, 64:320].contiguous(), su)
    assert want.shape == (4, 3, 57) and want.dtype == torch.bfloat16
    assert torch.equal(dense.int8_gated_matmul(codes[:, ::2, 16:272], scale[:, ::2], wg[:, :256], sg, wu[:, 64:320], su), want)
    one = dense.int8_gated_matmul(codes[0, 0], scale[0, 0], wg, sg, wu, su, out_dtype=torch.float16)
    assert one.shape == (57,) and torch.equal(one, dense.int8_gated_matmul(codes[0], scale[0], wg, sg, wu, su, torch.float16)[0])
    assert dense.int8_gated_matmul(codes[:0], scale[:0], wg, sg, wu, su).shape == (0, 6, 57)
    for bad in ((codes.float(), scale, wg, sg, wu, su), (codes, scale.half(), wg, sg, wu, su), (codes, scale, wg.float(), sg, wu, su),
                (codes, scale, wg, sg, wu, su, torch.float32)):
        with pytest.raises(TypeError):
            dense.int8_gated_matmul(*bad)
    for bad in ((codes, scale[:1], wg, sg, wu, su), (codes, scale.cpu(), wg, sg, wu, su), (codes, scale, wg[:-1], sg[:-1], wu, su),
                (codes, scale, wg, sg[:-1], wu, su), (codes[..., :256], scale, wg, sg, wu, su), (codes[..., :100], scale, wg, sg, wu, su)):
        with pytest.raises(ValueError):
            dense.int8_gated_matmul(*bad)
    with pytest.raises(_lib.DmoqError):
        dense.int8_gated_matmul(codes.cpu(), scale.cpu(), wg, sg, wu, su)


@pytest.mark.parametrize("t", (1, 12, 40, 200, 2500))
def test_gates_far_below_zero(t):
    """silu(g) down to g = -95, where the sigmoid is a subnormal 32-bit number; an up value of 1e6 brings it back."""
    n = 400
    x = torch.zeros(t, 16, dtype=torch.bfloat16, device=DEV)
    x[:, 0] = 127.0                                                  # code 127, scale 1
    w = torch.zeros(n, 16, dtype=torch.int8, device=DEV)
    w[:, 0] = 127
    gate_scale = (-torch.linspace(0.0, 95.0, n) / 127 ** 2).to(DEV)
    h = dense.int8_gated_linear(x, w, gate_scale, w, torch.full((n,), 1e6 / 127 ** 2, device=DEV))
    gate, up = gate_scale.double().cpu() * 127 ** 2, float(torch.tensor(1e6 / 127 ** 2)) * 127 ** 2
    want = R.silu(gate) * up
    # relative: g carries two roundings, with silu's condition 1 + |g|, u two, the exponential 2 + 1.173 |g| units of 2^-23, five
    # more; absolute: the sigmoid and g times it are held to a unit of 2^-149
    e32 = 2.0 ** -24 * (2 * (1 + gate.abs()) + 2 + 2 * (2 + 1.173 * gate.abs()) + 5)
    tol = want.abs() * (2.0 ** -8 * (1 + e32) + e32) + up * (2 * gate.abs() + 1) * 2.0 ** -149
    assert ((h.double().cpu() - want).abs() <= tol).all()


def test_int8_shapes_strides_and_refusals():
    g = rng(11)
    x = randn(g, 4, 6, 512, dtype=torch.bfloat16)
    w, ws = weight8(g, 48, 256)
    y = dense.int8_linear(x[:, ::2, 128:384], w, ws)
    assert y.shape == (4, 3, 48) and torch.equal(y, dense.int8_linear(x[:, ::2, 128:384].contiguous(), w, ws))
    wide, wide_scale = weight8(g, 48, 512)
    assert torch.equal(dense.int8_linear(x[0, :, :256], wide[:, :256], ws), dense.int8_linear(x[0, :, :256], wide[:, :256].contiguous(), ws))
    assert dense.int8_linear(x[:0, 0, :256], w, ws).shape == (0, 48)
    assert dense.int8_linear(x[0, 0, :256], w, ws).shape == (48,)
    codes, s = dense.quantize_int8_tokens(x)
    part = dense.int8_matmul(codes[:, :, 16:272], s, w, ws)
    assert torch.equal(part, dense.int8_matmul(codes[:, :, 16:272].contiguous(), s, w, ws))
    with pytest.raises(TypeError):
        dense.int8_linear(x.float(), w, ws)
    with pytest.raises(TypeError):
        dense.int8_linear(x[..., :256], w, ws.half())
    with pytest.raises(TypeError):
        dense.int8_linear(x[..., :256], w, ws, torch.zeros(48, device=DEV))
    with pytest.raises(ValueError):
        dense.int8_linear(x, w, ws)                                  # inner sizes differ
    with pytest.raises(ValueError):
        dense.int8_linear(x[..., :256], w, ws[:-1])
    with pytest.raises(ValueError):
        dense.int8_linear(x[..., :256], w.cpu(), ws)
    with pytest.raises(ValueError):
        dense.quantize_int8_tokens(x[..., :100])
    with pytest.raises(ValueError):
        dense.int8_gated_linear(x[..., :256], w, ws, w[:-1], ws[:-1])
    with pytest.raises(TypeError):
        dense.int8_matmul(codes, s, wide, wide_scale, out_dtype=torch.float32)


# --------------------------------------------------------------------------------------------- gated feed-forward

FFN_SIZES = [(1, 8, 8), (1, 256, 136), (3, 72, 200), (16, 512, 256), (33, 128, 1032), (31, 1032, 264), (64, 256, 72), (100, 264, 2056), (128, 320, 128), (129, 264, 136),
             (257, 1032, 520), (1000, 256, 128), (640, 520, 1040), (1500, 1032, 1544),
             (9, 1032, 264), (2, 2056, 4104), (12, 2056, 4104), (200, 264, 1032), (256, 1032, 136)]


def ffn_inputs(t, h, i, dtype, seed=0):
    g = rng(seed + 7 * t + h + i)
    x = randn(g, t, h, dtype=dtype)
    wg, wu = (randn(g, i, h, scale=1.5 * h ** -0.5, dtype=dtype) for _ in range(2))
    wd = randn(g, h, i, scale=i ** -0.5, dtype=dtype)
    return x, wg, wu, wd, randn(g, t, h, dtype=dtype)


# y: hidden values and y rounded.  dw_down: hidden values and the gradient.  The others: dg or du, and the gradient.
ROUNDINGS = {"y": 2, "dx": 2, "dw_gate": 2, "dw_up": 2, "dw_down": 2}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,h,i", FFN_SIZES)
def test_ffn_forward(t, h, i, dtype):
    x, wg, wu, wd, _ = ffn_inputs(t, h, i, dtype)
    y = dense.gated_feed_forward(x, wg, wu, wd)
    assert not y.requires_grad
    R.close(y, R.ffn(x, wg, wu, wd)[3], ROUNDINGS["y"], "y")
    assert torch.equal(y, dense.gated_feed_forward(x, wg, wu, wd))
    healthy()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,h,i", FFN_SIZES)
def test_ffn_gradients(t, h, i, dtype):
    x, wg, wu, wd, dy = ffn_inputs(t, h, i, dtype, seed=1)
    leaves = [v.requires_grad_(True) for v in (x, wg, wu, wd)]
    y = dense.gated_feed_forward(*leaves)
    grads = dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), torch.autograd.grad(y, leaves, dy, retain_graph=True)))
    want = R.ffn_grads(x, wg, wu, wd, dy)
    R.close(y, R.ffn(x, wg, wu, wd)[3], ROUNDINGS["y"], "y")
    for name, v in grads.items():
        R.close(v, want[name], ROUNDINGS[name], name)
    again = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads.values(), again))
    healthy()


@pytest.mark.parametrize("dtype", DTYPES)
def test_ffn_gradients_against_differences(dtype):
    x, wg, wu, wd, dy = ffn_inputs(40, 136, 264, dtype, seed=2)
    leaves = [v.requires_grad_(True) for v in (x, wg, wu, wd)]
    grads = torch.autograd.grad(dense.gated_feed_forward(*leaves), leaves, dy)
    base = [v.detach().double().cpu() for v in leaves]
    g = rng(5)
    for i, grad in enumerate(grads):
        # along the gradient itself, so that the slope is its squared norm and nothing cancels
        way = grad.double().cpu() + 0.3 * grad.double().cpu().std() * torch.randn(grad.shape, generator=g).double()
        eps = 1e-5 / float(way.abs().max())
        loss = lambda e: float((R.ffn(*[b + (e * way if j == i else 0) for j, b in enumerate(base)])[3] * dy.double().cpu()).sum())  # noqa: E731
        slope = (loss(eps) - loss(-eps)) / (2 * eps)
        mine = float((grad.double().cpu() * way).sum())
        assert abs(mine - slope) <= 2 * R.half(dtype) * abs(slope) + 1e-6 * abs(slope), (i, mine, slope)


def test_ffn_computes_only_the_gradients_that_are_needed():
    x, wg, wu, wd, dy = ffn_inputs(70, 264, 136, torch.bfloat16, seed=3)
    want = R.ffn_grads(x, wg, wu, wd, dy)
    names = ("dx", "dw_gate", "dw_up", "dw_down")
    for mask in range(1, 16):
        leaves = [v.detach().clone().requires_grad_(bool(mask >> i & 1)) for i, v in enumerate((x, wg, wu, wd))]
        y = dense.gated_feed_forward(*leaves)
        y.backward(dy)
        for i, v in enumerate(leaves):
            assert (v.grad is None) == (not mask >> i & 1)
            if v.grad is not None:
                R.close(v.grad, want[names[i]], ROUNDINGS[names[i]], f"{names[i]} (mask {mask})")


@pytest.mark.parametrize("t", (3, 12, 70, 300, 2000))
def test_weights_that_are_parts_of_larger_matrices(t):
    """Row pitches of the weights (a shard of the columns of a matrix, halves of a joined one) in every kernel."""
    g = rng(40 + t)
    x, (w, ws), (w2, ws2) = acts(g, t, 528, torch.bfloat16), weight8(g, 1050, 1056), weight8(g, 1050, 544)
    a, b = w[:, 16:544], w2[:, :528]
    assert torch.equal(dense.int8_linear(x, a, ws), dense.int8_linear(x, a.contiguous(), ws))
    assert torch.equal(dense.int8_gated_linear(x, a, ws, b, ws2), dense.int8_gated_linear(x, a.contiguous(), ws, b.contiguous(), ws2))
    codes, scale = dense.quantize_int8_tokens(x)
    assert torch.equal(dense.int8_matmul(codes, scale, a, ws), dense.int8_linear(x, a, ws))
    joined = randn(g, 2 * 520, 544, scale=0.05, dtype=torch.bfloat16).requires_grad_(True)
    down = randn(g, 528, 1040, scale=0.05, dtype=torch.bfloat16).requires_grad_(True)
    x.requires_grad_(True)
    dy = randn(g, t, 528, dtype=torch.bfloat16)
    views = joined[:520, 8:536], joined[520:, 8:536], down[:, 512:1032]
    y = dense.gated_feed_forward(x, *views)
    dx, dj, dd = torch.autograd.grad(y, (x, joined, down), dy)
    flat = [v.detach().contiguous().requires_grad_(True) for v in views]
    want = dense.gated_feed_forward(x, *flat)
    grads = torch.autograd.grad(want, [x] + flat, dy)
    assert torch.equal(y, want) and torch.equal(dx, grads[0])
    assert torch.equal(dj[:, 8:536], torch.cat(grads[1:3])) and torch.equal(dd[:, 512:1032], grads[3])
    R.close(y, R.ffn(x, *flat)[3], ROUNDINGS["y"], "y")


def test_ffn_gradients_of_shared_and_broadcast_arguments():
    """One weight for both projections; a token repeated without memory of its own; a weight of repeated rows."""
    _, wg, wu, wd, dy = ffn_inputs(50, 136, 264, torch.bfloat16, seed=13)
    token = randn(rng(14), 1, 136, dtype=torch.bfloat16).requires_grad_(True)
    row = randn(rng(15), 1, 136, scale=0.1, dtype=torch.bfloat16).requires_grad_(True)
    w, wd = wg.requires_grad_(True), wd.requires_grad_(True)
    x = token.expand(50, 136)
    for gate, up in ((w, w), (row.expand(264, 136), w)):
        leaves = [token, w, wd] + ([row] if gate is not w else [])
        grads = torch.autograd.grad(dense.gated_feed_forward(x, gate, up, wd), leaves, dy)
        want = R.ffn_grads(x, gate, up, wd, dy)
        # sums over 50 tokens or 264 rows of gradients that were rounded once: one more rounding of the sum itself
        R.close(grads[0], want["dx"].sum(0, keepdim=True), ROUNDINGS["dx"] + 1, "token")
        R.close(grads[1], want["dw_gate"] + want["dw_up"] if gate is w else want["dw_up"], ROUNDINGS["dw_up"] + 1, "weight")
        R.close(grads[2], want["dw_down"], ROUNDINGS["dw_down"], "dw_down")
        if gate is not w:
            R.close(grads[3], want["dw_gate"].sum(0, keepdim=True), ROUNDINGS["dw_gate"] + 1, "row")


def test_ffn_empty_shapes_strides_and_refusals():
    x, wg, wu, wd, dy = ffn_inputs(24, 264, 136, torch.float16, seed=4)
    leaves = [v.requires_grad_(True) for v in (x[:0].detach(), wg, wu, wd)]
    y = dense.gated_feed_forward(*leaves)
    assert y.shape == (0, 264)
    gx, *gw = torch.autograd.grad(y.sum(), leaves)
    assert gx.shape == (0, 264) and all(float(v.abs().max()) == 0 for v in gw)
    # a view of a wider tensor, three dimensions, an upstream gradient without memory of its own
    wide = randn(rng(5), 4, 6, 400, dtype=torch.float16).requires_grad_(True)
    view = wide[:, 1:5, 64:328]
    gy = torch.autograd.grad(dense.gated_feed_forward(view, wg, wu, wd).sum(), (wide, wg))
    flat = view.detach().reshape(-1, 264).contiguous().requires_grad_(True)
    out = dense.gated_feed_forward(flat, wg, wu, wd)
    gf = torch.autograd.grad(out, (flat, wg), torch.ones_like(out))
    assert torch.equal(gy[0][:, 1:5, 64:328].reshape(-1, 264), gf[0]) and torch.equal(gy[1], gf[1])
    assert float(gy[0][:, 0].abs().max()) == 0
    # weights that are views
    assert torch.equal(dense.gated_feed_forward(x.detach(), wg.t().contiguous().t(), wu, wd), dense.gated_feed_forward(x.detach(), wg, wu, wd))
    with pytest.raises(TypeError):
        dense.gated_feed_forward(x, wg.bfloat16(), wu, wd)
    with pytest.raises(ValueError):
        dense.gated_feed_forward(x, wg, wu[:-8], wd)
    with pytest.raises(ValueError):
        dense.gated_feed_forward(x, wg, wu, wd.t())
    with pytest.raises(ValueError):
        dense.gated_feed_forward(x[:, :260], wg[:, :260], wu[:, :260], wd[:260])
    with pytest.raises(ValueError):
        dense.gated_feed_forward(x, wg, wu, wd.cpu())
    double = torch.autograd.grad(dense.gated_feed_forward(x, wg, wu, wd).square().sum(), wg, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        double.sum().backward()                                      # once differentiable


def test_ffn_sizes_beyond_the_limits_are_refused_before_any_work():
    """One token or one element each in memory: the sizes are those of views."""
    w = torch.zeros(8, 8, dtype=torch.bfloat16, device=DEV)
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device=DEV)
    for leaf in (x, w):
        leaf.requires_grad_(True)
        with pytest.raises(ValueError, match="2\\^26"):
            dense.gated_feed_forward(x.expand((1 << 26) + 1, 8), w, w, w)
        leaf.requires_grad_(False)
    one = torch.zeros(1, dtype=torch.bfloat16, device=DEV)
    for h, i in (((1 << 29) + 8, 8), (8, (1 << 29) + 8)):
        with pytest.raises(ValueError, match="2\\^29"):
            dense.gated_feed_forward(one.expand(1, h), one.expand(i, h), one.expand(i, h), one.expand(h, i))


def test_ffn_second_derivatives_raise_whatever_the_loss_is():
    """A gradient of a gradient must never be left out in silence, also where the upstream gradient is a constant."""
    x, wg, wu, wd, dy = ffn_inputs(24, 264, 136, torch.bfloat16, seed=16)
    leaves = [v.requires_grad_(True) for v in (x, wg, wu, wd)]
    want = torch.autograd.grad(dense.gated_feed_forward(*leaves), leaves, dy)
    for loss in (lambda y: y.sum(), lambda y: (y * dy).sum(), lambda y: y.float().square().sum()):
        y = dense.gated_feed_forward(*leaves)
        g = torch.autograd.grad(loss(y), leaves, create_graph=True)
        assert all(v.requires_grad for v in g)
        for v in g:
            with pytest.raises(RuntimeError, match="differentiable once"):
                (loss(dense.gated_feed_forward(*leaves)) + v.float().square().sum()).backward()
        for v in leaves:
            v.grad = None
    # the gradients themselves are what they are without a graph of them
    g = torch.autograd.grad(dense.gated_feed_forward(*leaves), leaves, dy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(g, want))
    # only some arguments
    frozen = [x.detach(), wg, wu.detach(), wd.detach()]
    g, = torch.autograd.grad(dense.gated_feed_forward(*frozen).sum(), wg, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.float().sum().backward()


@pytest.mark.parametrize("which", range(4))
def test_ffn_forward_mode_is_refused(which):
    """A tangent must not be dropped in silence, whether or not a gradient is asked for as well."""
    import torch.autograd.forward_ad as fwad

    args = list(ffn_inputs(24, 264, 136, torch.bfloat16, seed=17)[:4])
    with fwad.dual_level():
        assert not dense.gated_feed_forward(*args).requires_grad     # no tangents: as ever
        args[which] = fwad.make_dual(args[which], torch.ones_like(args[which]))
        for grad in (False, True):
            plain = [v if i == which else v.detach().requires_grad_(grad) for i, v in enumerate(args)]
            with pytest.raises(NotImplementedError):
                dense.gated_feed_forward(*plain)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                dense.gated_feed_forward(*plain)
    fn = lambda v: dense.gated_feed_forward(v, *args[1:])            # noqa: E731
    if which == 0:
        x = ffn_inputs(24, 264, 136, torch.bfloat16, seed=17)[0]
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(fn, (x,), (torch.ones_like(x),))


def test_ffn_with_saved_tensors_moved_and_from_other_threads():
    """What is saved may come back from a hook laid out anew; calls may come from several threads and streams at once."""
    import threading

    x, wg, wu, wd, dy = ffn_inputs(90, 264, 136, torch.bfloat16, seed=8)
    wide = torch.zeros(90, 400, dtype=torch.bfloat16, device=DEV)
    wide[:, 64:328] = x
    leaves = [wide[:, 64:328].requires_grad_(True)] + [v.requires_grad_(True) for v in (wg, wu, wd)]
    want = torch.autograd.grad(dense.gated_feed_forward(*leaves), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = dense.gated_feed_forward(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))
    results = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            mine = [v.detach().clone().requires_grad_(True) for v in leaves]
            for _ in range(10):
                results[i] = torch.autograd.grad(dense.gated_feed_forward(*mine), mine, dy)
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_ffn_infinities_and_nan_stay_in_their_rows():
    x, wg, wu, wd, _ = ffn_inputs(140, 264, 136, torch.bfloat16, seed=6)
    clean = dense.gated_feed_forward(x, wg, wu, wd)
    x2 = x.clone()
    x2[3, 5], x2[131, 0] = float("nan"), float("inf")
    y = dense.gated_feed_forward(x2, wg, wu, wd)
    rest = [r for r in range(140) if r not in (3, 131)]
    assert torch.equal(y[rest], clean[rest]) and torch.isnan(y[3]).all() and not torch.isfinite(y[131]).any()


# --------------------------------------------------------------------------------------------- how they are used

def test_outputs_stay_inside_their_memory():
    """Through the C entries, with rows of sentinels in front of and behind every output."""
    lib = _lib.load()
    for t, n, k in ((5, 37, 128), (130, 129, 256), (200, 1001, 128)):
        g = rng(n)
        x, (w, ws) = acts(g, t, k, torch.bfloat16), weight8(g, n, k)
        out = torch.full((t + 2, n), 7.0, dtype=torch.bfloat16, device=DEV)
        need = max(int(lib.dmoq_int8_scratch_bytes(t, n, k, 0)), int(lib.dmoq_int8_scratch_bytes(t, n, k, 1)), 16)
        scratch = torch.full((need + 256,), 99, dtype=torch.uint8, device=DEV)
        p = lambda v: C.c_void_p(v.data_ptr())  # noqa: E731
        for name, extra in (("dmoq_int8_linear", (p(w), k, p(ws), None)), ("dmoq_int8_gated_linear", (p(w), k, p(ws), p(w), k, p(ws)))):
            _lib.check(getattr(lib, name)(p(x), 1, k, *extra, t, n, k, p(scratch[128:]), p(out[1]), None), name)
            torch.cuda.synchronize()
            assert (out[0] == 7.0).all() and (out[-1] == 7.0).all() and torch.isfinite(out).all()
            assert (scratch[:128] == 99).all() and (scratch[128 + need:] == 99).all()
    t, h, i = 130, 136, 72
    x, wg, wu, wd, dy = ffn_inputs(t, h, i, torch.bfloat16)
    pad = lambda r, c: torch.full((r + 2, c), 7.0, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    hid, saved, y = pad(t, i), pad(3 * t, i), pad(t, h)
    dgu, dx, dw, dwd = pad(t, 2 * i), pad(t, h), pad(2 * i, h), pad(h, i)
    q = lambda v: C.c_void_p(v[1].data_ptr())  # noqa: E731
    _lib.check(lib.dmoq_gated_ffn(p(x), 1, h, p(wg), h, p(wu), h, p(wd), i, t, h, i, q(hid), i, q(saved), q(y), None), "ffn")
    _lib.check(lib.dmoq_gated_ffn_backward(p(dy), h, p(x), 1, h, p(wg), h, p(wu), h, p(wd), i, t, h, i, q(hid), i, q(saved), q(dgu), 2 * i, q(dx), q(dw),
                                           C.c_void_p(dw[1 + i].data_ptr()), q(dwd), None), "ffn backward")
    torch.cuda.synchronize()
    for v in (hid, saved, y, dgu, dx, dw, dwd):
        assert (v[0] == 7.0).all() and (v[-1] == 7.0).all()
    R.close(dw[1:1 + 2 * i], torch.cat([R.ffn_grads(x, wg, wu, wd, dy)[k] for k in ("dw_gate", "dw_up")]), 2, "dw")
    # the gradients of the two projections in memory that is not adjacent: two products
    a, b = pad(i, h), pad(i, h)
    _lib.check(lib.dmoq_gated_ffn_backward(p(dy), h, p(x), 1, h, None, 0, None, 0, p(wd), i, t, h, i, None, 0, q(saved), q(dgu), 2 * i, None, q(a), q(b),
                                           None, None), "ffn backward")
    torch.cuda.synchronize()
    assert torch.equal(a[1:-1], dw[1:1 + i]) and torch.equal(b[1:-1], dw[1 + i:1 + 2 * i])
    assert (a[-1] == 7.0).all() and (b[0] == 7.0).all()


def test_streams_and_captured_graphs():
    """Work goes to the current stream; two captured graphs replayed at once do not share scratch."""
    g = rng(21)
    k, n = 512, 640
    w, ws = weight8(g, n, k)
    xs = [acts(g, t, k, torch.bfloat16) for t in (40, 300)]
    fx, wg, wu, wd, _ = ffn_inputs(300, 264, 136, torch.bfloat16, seed=9)

    def work(x):
        return dense.int8_linear(x, w, ws), dense.int8_gated_linear(x, w, ws, w, ws), dense.gated_feed_forward(fx, wg, wu, wd)

    want = [[v.clone() for v in work(x)] for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)                                # whatever ran on another stream would be too early
        late = [x.clone() for x in xs]
        got = [work(x) for x in late]
    side.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs, static, outs = [], [torch.zeros_like(x) for x in xs], []
    for s in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(s))
        graphs.append(graph)
    for s, x in zip(static, xs):
        s.copy_(x)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    healthy()


def test_capture_over_two_streams():
    """Kernels that may overlap their predecessor, captured across a fork and a join and among kernels of others."""
    g = rng(22)
    x, (w, ws) = acts(g, 200, 512, torch.bfloat16), weight8(g, 512, 512)
    fx, wg, wu, wd, _ = ffn_inputs(3000, 512, 640, torch.bfloat16, seed=10)

    def work(side):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        a = dense.int8_linear(x, w, ws)
        with torch.cuda.stream(side):
            b = dense.gated_feed_forward(fx, wg, wu, wd)
            c = dense.gated_feed_forward(b[:7] * 0.5, wg, wu, wd)
        a = dense.int8_linear(a + 1, w, ws)
        main.wait_stream(side)
        return dense.int8_linear(a + b[:200], w, ws), dense.gated_feed_forward(c, wg, wu, wd)

    side = torch.cuda.Stream()
    want = [v.clone() for v in work(side)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(side)
    for _ in range(3):
        for v in got:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_training_step_in_a_captured_graph():
    x, wg, wu, wd, dy = ffn_inputs(96, 264, 136, torch.bfloat16, seed=12)
    leaves = [v.requires_grad_(True) for v in (x, wg, wu, wd)]

    def step():
        return torch.autograd.grad(dense.gated_feed_forward(*leaves), leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [v.clone() for v in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for v in got:
        v.fill_(0)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("tokens", (1, 40, 700))
@pytest.mark.parametrize("eight_bit", (False, True))
def test_as_shared_expert_of_a_packed_layer(tokens, eight_bit):
    """The MoE module with an unpacked shared expert: routed experts packed, the shared one a dense block of this file."""
    moe = synth.build_layer(hidden=256, n_experts=8, top_k=2, inter=128, bit_mix={2: 0.5, 4: 0.5}, seed=5).to(DEV)
    x = synth.make_activations(tokens, 256, seed=3).to(DEV).unsqueeze(0)
    routed = moe(x).clone()
    g = rng(tokens)
    block = D.GatedFeedForward(256, 384, device=DEV)
    with torch.no_grad():
        for p in block.parameters():
            p.copy_(randn(g, *p.shape, scale=0.05, dtype=torch.bfloat16))
    expert = D.W8A8GatedFeedForward.from_mlp(block) if eight_bit else block
    moe.shared_expert = expert
    moe.shared_expert_gate = torch.nn.Linear(256, 1, bias=False, dtype=torch.bfloat16, device=DEV)
    for _ in range(3):                                              # eager, captured, replayed
        y = moe(x)
        want = routed[0] + expert(x[0]) * torch.sigmoid(moe.shared_expert_gate(x[0]))
        assert torch.equal(y[0], want)
    ref = R.ffn(x[0], block.gate_proj.weight, block.up_proj.weight, block.down_proj.weight)[3]
    if eight_bit:
        # two quantisations of tokens and one of every weight: each is off by at most half a step, max / 254, of a row whose
        # root mean square is at least max / 127 * 10 here, and rounding errors of a row add up in squares (x 1 / sqrt(3))
        assert float((expert(x[0]).double().cpu() - ref).norm() / ref.norm()) <= 4 * 0.5 / 10 / 3 ** 0.5
    else:
        R.close(expert(x[0]), ref, 2, "shared expert")
    healthy()


@pytest.mark.parametrize("dtype", DTYPES)
def test_modules(dtype):
    g = rng(31)
    lin = torch.nn.Linear(144, 57, bias=True, dtype=dtype, device=DEV)
    q = D.W8A8Linear.from_linear(lin)
    codes, s = R.quantize(lin.weight)
    assert torch.equal(q.weight.double().cpu(), codes) and torch.equal(q.weight_scale.cpu(), s.float())
    x = acts(g, 9, 144, dtype)
    assert torch.equal(q(x), dense.int8_linear(x, q.weight, q.weight_scale, q.bias))
    again = D.W8A8Linear.from_metadata({"out_features": 57, "in_features": 144, "bias_shape": [57], "orig_dtype": str(dtype)})
    again.load_state_dict(q.state_dict(), strict=True, assign=True)
    assert torch.equal(again(x), q(x))
    block = D.GatedFeedForward(144, 72, dtype=dtype, device=DEV)
    y = block(x)
    y.float().square().sum().backward()
    grads = R.ffn_grads(x, *(p.weight for p in (block.gate_proj, block.up_proj, block.down_proj)), 2 * y)
    for p, name in ((block.gate_proj, "dw_gate"), (block.up_proj, "dw_up"), (block.down_proj, "dw_down")):
        R.close(p.weight.grad, grads[name], ROUNDINGS[name], name)


def test_int8_results_do_not_depend_on_the_batch():
    """A token's 8-bit results are the same in every kernel that its batch's size may select."""
    g = rng(77)
    k, n = 1040, 6000
    x, (w, ws), (w2, ws2) = acts(g, 5000, k, torch.bfloat16), weight8(g, n, k), weight8(g, n, k)
    b = randn(g, n, dtype=torch.bfloat16)
    lin, gated = dense.int8_linear(x, w, ws, b), dense.int8_gated_linear(x, w, ws, w2, ws2)
    for t in (1, 3, 8, 9, 16, 17, 40, 70, 129, 200, 300, 700, 1500):
        assert torch.equal(dense.int8_linear(x[:t], w, ws, b), lin[:t]), t
        assert torch.equal(dense.int8_gated_linear(x[:t], w, ws, w2, ws2), gated[:t]), t
        assert torch.equal(dense.int8_linear(x[:t], w[:500], ws[:500]), dense.int8_linear(x, w[:500], ws[:500])[:t]), t


@pytest.mark.filterwarnings("ignore")
def test_modules_refuse_to_be_traced():
    block = D.GatedFeedForward(144, 80, device=DEV)
    x = randn(rng(60), 5, 144, dtype=torch.bfloat16)
    for module in (block, D.W8A8GatedFeedForward.from_mlp(block), D.W8A8Linear.from_linear(block.gate_proj)):
        with pytest.raises(_lib.DmoqError, match="traced"):
            torch.jit.trace(module, (x,))
        assert torch.isfinite(module(x)).all()                       # and run as ever afterwards


FIRST_USE = """
import sys
sys.path.insert(0, %r)
import torch
from dartmoq_b200 import dense
torch.manual_seed(0)
w, s = torch.randint(-100, 100, (640, 512), device="cuda", dtype=torch.int8), torch.rand(640, device="cuda")
f = [torch.randn(640, 512, device="cuda").bfloat16() * 0.05 for _ in range(2)] + [torch.randn(512, 640, device="cuda").bfloat16() * 0.05]
xs = [torch.randn(t, 512, device="cuda").bfloat16() for t in (4, 40, 300, 3000)]
work = lambda x: (dense.int8_linear(x, w, s), dense.int8_gated_linear(x, w, s, w, s), dense.gated_feed_forward(x, *f))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = [work(x) for x in xs]
graph.replay()
torch.cuda.synchronize()
for x, g in zip(xs, got):
    assert all(torch.equal(a, b) for a, b in zip(work(x), g)), x.shape
print("same")
"""


def test_first_use_inside_a_capture():
    """A fresh process whose first call of every kernel is made while a stream is being captured."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_USE % root], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]


FIRST_USE_BY_THREADS = """
import sys, threading
sys.path.insert(0, %r)
import torch
from dartmoq_b200 import dense
torch.manual_seed(0)
w, s = torch.randint(-100, 100, (640, 512), device="cuda", dtype=torch.int8), torch.rand(640, device="cuda")
f = [torch.randn(640, 512, device="cuda").bfloat16() * 0.05 for _ in range(2)] + [torch.randn(512, 640, device="cuda").bfloat16() * 0.05]
xs = [torch.randn(t, 512, device="cuda").bfloat16() for t in (4, 40, 300, 3000)]
work = lambda x: (dense.int8_linear(x, w, s), dense.int8_gated_linear(x, w, s, w, s), dense.gated_feed_forward(x, *f))
torch.cuda.synchronize()
start, got = threading.Barrier(8), [None] * 8

def first(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        got[i] = [work(x) for x in xs]
        torch.cuda.current_stream().synchronize()

threads = [threading.Thread(target=first, args=(i,)) for i in range(8)]
for t in threads:
    t.start()
for t in threads:
    t.join()
for g in got:
    assert all(torch.equal(a, b) for x, o in zip(xs, g) for a, b in zip(work(x), o))
print("same")
"""


def test_first_use_by_several_threads_at_once():
    """A fresh process in which eight threads make the first call of every kernel together."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_USE_BY_THREADS % root], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "same", r.stderr[-2000:]

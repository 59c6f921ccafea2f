"""Dense operators, what needs no GPU: refusals of the C entry points and of the Python functions, module plumbing."""
import ctypes as C

import pytest
import torch

import dartmoq_b200 as D
from dartmoq_b200 import _lib, dense

EINVAL, ESIZE, OK = -1, -3, 0
P = C.c_void_p(4096)          # an aligned address that no refused call touches
ODD = C.c_void_p(4104)        # not 16-byte aligned


def test_token_quant_refuses():
    f = _lib.load().dmoq_token_quant
    assert f(P, 1, 0, 128, 128, P, P, None) == OK                    # no tokens: nothing to do
    for bad in ((None, 1, 4, 128, 128, P, P), (P, 1, 4, 128, 128, None, P), (P, 1, 4, 128, 128, P, None),
                (ODD, 1, 4, 128, 128, P, P), (P, 1, 4, 128, 128, ODD, P),
                (P, 1, 4, 120, 120, P, P), (P, 1, 4, 0, 0, P, P), (P, 1, -1, 128, 128, P, P),
                (P, 1, 4, 128, 124, P, P), (P, 1, 4, 128, 132, P, P)):
        assert f(*bad, None) == EINVAL, bad


def each(f, good, want, bad):
    for i, v in bad:
        assert f(*(good[:i] + [v] + good[i + 1:]), None) == want, (i, v)


def test_int8_products_refuse():
    lib = _lib.load()
    #       codes scales w pitch scale bias bf16 T N K out
    good = [P, P, P, 128, P, None, 1, 4, 33, 128, P]
    each(lib.dmoq_int8_gemm, good, OK, [(7, 0)])
    each(lib.dmoq_int8_gemm, good, EINVAL, [(i, None) for i in (0, 1, 2, 4, 10)])
    each(lib.dmoq_int8_gemm, good, EINVAL, [(0, ODD), (2, ODD), (3, 112), (3, 136), (7, -1), (8, 0), (9, 8), (9, 0), (9, 136)])
    each(lib.dmoq_int8_gemm, good, ESIZE, [(9, 131072), (7, (1 << 30) + 1), (8, (1 << 30) + 1)])
    #       codes scales gate pitch scale up pitch scale bf16 T I K out
    good = [P, P, P, 128, P, P, 128, P, 1, 4, 33, 128, P]
    each(lib.dmoq_int8_gated_gemm, good, OK, [(9, 0)])
    each(lib.dmoq_int8_gated_gemm, good, EINVAL, [(i, None) for i in (0, 1, 2, 4, 5, 7, 12)] + [(3, 112), (6, 136), (2, ODD), (5, ODD)])
    each(lib.dmoq_int8_gated_gemm, good, ESIZE, [(11, 1 << 20)])
    # with the quantiser in front nothing is launched before everything is known to be right
    #       x bf16 pitch w pitch scale bias T N K scratch out
    good = [P, 1, 128, P, 128, P, None, 40, 33, 128, P, P]
    each(lib.dmoq_int8_linear, good, EINVAL, [(0, None), (2, 127), (3, None), (4, 100), (5, None), (8, 0), (9, 100), (10, None), (11, None),
                                              (3, ODD), (10, ODD)])
    each(lib.dmoq_int8_linear, good, ESIZE, [(9, 131072)])
    #       x bf16 pitch gate pitch scale up pitch scale T I K scratch out
    good = [P, 1, 128, P, 128, P, P, 128, P, 40, 33, 128, P, P]
    each(lib.dmoq_int8_gated_linear, good, EINVAL, [(i, None) for i in (0, 3, 5, 6, 8, 12, 13)] + [(4, 120), (7, 96)])


def test_int8_scratch_size():
    f = _lib.load().dmoq_int8_scratch_bytes
    assert f(40, 33, 128, 0) == 40 * 128 + 40 * 4 and f(1000, 1, 131056, 1) == 1000 * 131072 + 4000   # whole 128-byte lines
    assert f(0, 33, 128, 0) == 0 and f(1, 33, 128, 1) == 0 and f(8, 512, 1024, 0) == 0   # none; few: the product makes the codes
    assert f(8, 64, 8192, 0) == 8 * 8192 + 32 and f(1, 8, 65536, 0) == 65536 + 4         # few, but too long for that
    assert f(1, 16384, 1024, 0) == 0 and f(20, 8, 16, 1) == 20 * 132 and f(1, 16400, 1024, 0) == 1028 and f(1, 16384, 1024, 1) == 1028   # or too many blocks
    assert f(9, 33, 128, 0) == 9 * 128 + 36
    assert f(4, 33, 100, 0) == 0 and f(-1, 33, 128, 0) == 0                              # refused by the calls themselves


def test_gated_ffn_refuses():
    lib = _lib.load()
    #       x bf pitch wg  p   wu  p   wd  p   T  H   I   h  p   saved y
    good = [P, 1, 64, P, 64, P, 64, P, 32, 4, 64, 32, P, 64, None, P]
    each(lib.dmoq_gated_ffn, good, OK, [(9, 0)])
    each(lib.dmoq_gated_ffn, good, EINVAL, [(i, v) for i in (0, 3, 5, 7, 12, 15) for v in (None, ODD)] + [(14, ODD)])
    each(lib.dmoq_gated_ffn, good, EINVAL, [(2, 60), (2, 68), (4, 56), (6, 68), (8, 24), (13, 24), (13, 36), (10, 60), (10, 0), (11, 12), (11, 0),
                                            (9, -4)])
    each(lib.dmoq_gated_ffn, good, ESIZE, [(10, (1 << 29) + 8), (11, (1 << 29) + 8)])
    #       dy p  x bf p  wg  p   wu  p   wd  p   T  H   I   h  p saved dgu p dx dwg dwu dwd
    good = [P, 64, P, 1, 64, P, 64, P, 64, P, 32, 4, 64, 32, P, 32, P, P, 64, P, P, P, P]
    each(lib.dmoq_gated_ffn_backward, good, EINVAL, [(i, v) for i in (0, 2, 5, 7, 9, 14, 16, 17) for v in (None, ODD)])
    each(lib.dmoq_gated_ffn_backward, good, EINVAL, [(19, ODD), (20, ODD), (22, ODD), (1, 60), (4, 60), (6, 56), (8, 68), (10, 24), (12, 4),
                                                     (13, 12), (15, 24), (18, 56), (18, 68)])
    each(lib.dmoq_gated_ffn_backward, good, ESIZE, [(11, (1 << 26) + 1)])


def test_functions_refuse_cpu_tensors():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w8, s8 = torch.zeros(32, 64, dtype=torch.int8), torch.zeros(32)
    w = torch.zeros(32, 64, dtype=torch.bfloat16)
    for call in (lambda: dense.quantize_int8_tokens(x), lambda: dense.int8_linear(x, w8, s8),
                 lambda: dense.int8_gated_linear(x, w8, s8, w8, s8), lambda: dense.gated_feed_forward(x, w, w, w.t()),
                 lambda: dense.int8_matmul(w8, s8, w8, s8), lambda: D.GatedFeedForward(64, 32)(x)):
        with pytest.raises(_lib.DmoqError):
            call()


@pytest.mark.parametrize("k", ((1 << 32) + 16, (1 << 31), (1 << 30) + 16))
def test_inner_sizes_past_32_bits_are_refused(k):
    with pytest.raises(ValueError, match="2\\^30"):
        dense._check_k8(k)


def test_functions_refuse_to_be_traced():
    """A recorded call would return memory that nothing fills."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w8, s8 = torch.zeros(32, 64, dtype=torch.int8), torch.zeros(32)
    w = torch.zeros(32, 64, dtype=torch.bfloat16)
    for call in (dense.quantize_int8_tokens, lambda v: dense.int8_linear(v, w8, s8), lambda v: dense.int8_gated_linear(v, w8, s8, w8, s8),
                 lambda v: dense.gated_feed_forward(v, w, w, w.t()), lambda v: dense.int8_matmul(v.to(torch.int8), s8[:4], w8, s8)):
        with pytest.raises(_lib.DmoqError, match="traced"):
            torch.jit.trace(call, (x,))
        with pytest.raises(_lib.DmoqError, match="traced"):
            make_fx(call)(x)


def test_tangents_are_seen():
    import torch.autograd.forward_ad as fwad

    x = torch.zeros(3)
    assert not dense._has_tangent(x)
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones(3))
        assert not dense._has_tangent(x) and dense._has_tangent(x, dual)
        with torch.no_grad():
            assert dense._has_tangent(dual)


def test_w8a8_linear_plumbing():
    lin = D.W8A8Linear.from_metadata({"out_features": 33, "in_features": 64, "bias_shape": [33], "orig_dtype": "torch.float16"})
    assert set(lin.state_dict()) == {"weight", "weight_scale", "bias"}
    src = {"weight": torch.randint(-127, 128, (33, 64), dtype=torch.int8), "weight_scale": torch.rand(33),
           "bias": torch.rand(33).half()}
    lin.load_state_dict(src, strict=True, assign=True)
    assert torch.equal(lin.weight, src["weight"]) and lin.bias.dtype == torch.float16
    lin.to(torch.bfloat16)                                           # the bias follows, the scales stay 32-bit
    assert lin.bias.dtype == torch.bfloat16 and torch.equal(lin.weight_scale, src["weight_scale"])
    assert set(D.W8A8Linear.from_metadata({"out_features": 3, "in_features": 16}).state_dict()) == {"weight", "weight_scale"}
    with pytest.raises(ValueError):
        D.W8A8Linear(torch.zeros(4, 24, dtype=torch.int8), torch.zeros(4))
    with pytest.raises(ValueError):
        D.W8A8Linear(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(5))
    with pytest.raises(TypeError):
        D.W8A8Linear(torch.zeros(4, 32), torch.zeros(4))


def test_feed_forward_plumbing():
    class Mlp(torch.nn.Module):
        def __init__(self, bias=False):
            super().__init__()
            self.gate_proj, self.up_proj = torch.nn.Linear(64, 32, bias=bias), torch.nn.Linear(64, 32, bias=bias)
            self.down_proj = torch.nn.Linear(32, 64, bias=bias)

    mlp = Mlp()
    block = D.GatedFeedForward.from_mlp(mlp)
    assert block.gate_proj is mlp.gate_proj and set(block.state_dict()) == set(mlp.state_dict())
    assert (block.hidden_size, block.intermediate_size) == (64, 32)
    assert {k: tuple(v.shape) for k, v in D.GatedFeedForward(64, 32).state_dict().items()} == \
        {"gate_proj.weight": (32, 64), "up_proj.weight": (32, 64), "down_proj.weight": (64, 32)}
    with pytest.raises(ValueError):
        D.GatedFeedForward.from_mlp(Mlp(bias=True))
    with pytest.raises(TypeError):
        D.GatedFeedForward.from_mlp(torch.nn.Linear(2, 2))
    lin = lambda n, k: D.W8A8Linear(torch.zeros(n, k, dtype=torch.int8), torch.zeros(n))   # noqa: E731
    assert set(D.W8A8GatedFeedForward(lin(32, 64), lin(32, 64), lin(64, 32)).state_dict()) == \
        {f"{p}_proj.{t}" for p in ("gate", "up", "down") for t in ("weight", "weight_scale")}
    with pytest.raises(ValueError):
        D.W8A8GatedFeedForward(lin(32, 64), lin(48, 64), lin(64, 32))
    with pytest.raises(ValueError):
        D.W8A8GatedFeedForward(lin(32, 64), lin(32, 64), lin(64, 48))


class Mlp(torch.nn.Module):
    def __init__(self, **attributes):
        super().__init__()
        self.gate_proj, self.up_proj = torch.nn.Linear(64, 32, bias=False), torch.nn.Linear(64, 32, bias=False)
        self.down_proj = torch.nn.Linear(32, 64, bias=False)
        for name, value in attributes.items():
            setattr(self, name, value)


class Doubled(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


def test_from_mlp_takes_silu_blocks():
    F = torch.nn.functional
    for act in (torch.nn.SiLU(), F.silu, lambda z: z * torch.sigmoid(z), "silu", "Swish"):
        for name in ("act_fn", "hidden_act"):
            assert D.GatedFeedForward.from_mlp(Mlp(**{name: act})).hidden_size == 64
    assert D.GatedFeedForward.from_mlp(Mlp(act=None, activation=0.5)).intermediate_size == 32     # not an activation


def test_from_mlp_refuses_what_it_would_compute_otherwise():
    F = torch.nn.functional
    for act in (torch.nn.GELU(), F.relu, "gelu", "gelu_pytorch_tanh", torch.nn.PReLU(), torch.nn.GLU(), lambda z: z, lambda a, b: a):
        for name in ("act_fn", "activation_fn", "act", "activation", "hidden_act"):
            for cls in (D.GatedFeedForward, D.W8A8GatedFeedForward):
                with pytest.raises(ValueError, match=name):
                    cls.from_mlp(Mlp(**{name: act}))
    for part in ("gate_proj", "up_proj", "down_proj"):
        mlp = Mlp(act_fn=torch.nn.SiLU())
        n, k = getattr(mlp, part).weight.shape
        setattr(mlp, part, Doubled(k, n, bias=False))
        with pytest.raises(ValueError, match="Doubled"):
            D.GatedFeedForward.from_mlp(mlp)
        for register in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"):
            mlp = Mlp()
            handle = getattr(getattr(mlp, part), register)(lambda *a: None)
            with pytest.raises(ValueError, match="hooks"):
                D.GatedFeedForward.from_mlp(mlp)
            handle.remove()
            D.GatedFeedForward.from_mlp(mlp)
        mlp = Mlp()
        getattr(mlp, part).forward = lambda x: x                     # as wrappers of a module's forward do
        with pytest.raises(ValueError):
            D.GatedFeedForward.from_mlp(mlp)
    mlp = Mlp()
    torch.nn.utils.parametrizations.weight_norm(mlp.up_proj)         # a computed weight is read as it is computed
    block = D.GatedFeedForward.from_mlp(mlp)
    assert block.up_proj.weight.grad_fn is not None

"""A layer's shared expert, its gate and its router assigned, replaced and removed between calls: eager, captured and replayed
calls always compute what the module holds now."""
import pytest
import torch

import dartmoq_b200 as D
from dartmoq_b200 import synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HIDDEN = 256


def layer(seed=5, **kw):
    return synth.build_layer(hidden=HIDDEN, n_experts=8, top_k=2, inter=128, bit_mix={2: 0.5, 4: 0.5}, seed=seed, **kw).to(DEV)


def block(seed):
    torch.manual_seed(seed)
    return D.GatedFeedForward(HIDDEN, 384, device=DEV)


def linear_gate(seed):
    torch.manual_seed(seed)
    return torch.nn.Linear(HIDDEN, 1, bias=False, dtype=torch.bfloat16, device=DEV)


def tokens(n=40):
    return synth.make_activations(n, HIDDEN, seed=3).to(DEV).unsqueeze(0)


def calls(moe, x, want):
    for _ in range(3):                              # eager, captured, replayed
        assert torch.equal(moe(x), want)


@torch.no_grad()
def with_dense(routed, x, expert, gate):
    return (routed[0] + expert(x[0]) * torch.sigmoid(gate(x[0]))).unsqueeze(0)


@pytest.mark.parametrize("n", (40, 700))
def test_dense_expert_and_gate_come_and_go(n):
    x, moe = tokens(n), layer()
    routed = moe(x).clone()
    calls(moe, x, routed)
    engine, a, b, ga, gb = moe._engine, block(1), block(2), linear_gate(3), linear_gate(4)
    moe.shared_expert = a
    calls(moe, x, routed)                           # no gate yet: the layer has no shared expert
    moe.shared_expert_gate = ga
    calls(moe, x, with_dense(routed, x, a, ga))
    moe.shared_expert_gate = gb
    calls(moe, x, with_dense(routed, x, a, gb))
    moe.shared_expert = b
    calls(moe, x, with_dense(routed, x, b, gb))
    moe.shared_expert_gate = None
    calls(moe, x, routed)
    moe.shared_expert, moe.shared_expert_gate = None, ga
    calls(moe, x, routed)
    moe.shared_expert = a
    calls(moe, x, with_dense(routed, x, a, ga))
    assert moe._engine is engine                    # the routed experts' weights were laid out once


@pytest.mark.parametrize("n", (40, 700))
def test_gates_replaced_after_a_capture(n):
    """The packed shared expert's gate and the router are part of the captured graph."""
    x = tokens(n)
    moe, fresh, other = layer(shared_inter=128), layer(shared_inter=128), layer(seed=6, shared_inter=128)
    first = moe(x).clone()
    calls(moe, x, first)
    gate = linear_gate(7)
    moe.shared_expert_gate = fresh.shared_expert_gate = gate
    want = fresh(x).clone()
    assert not torch.equal(want, first)
    calls(moe, x, want)
    moe.gate = other.gate
    fresh = layer(shared_inter=128)
    fresh.shared_expert_gate, fresh.gate = gate, other.gate
    again = fresh(x).clone()
    assert not torch.equal(again, want)
    calls(moe, x, again)


def test_packed_and_dense_experts_replace_one_another():
    x = tokens()
    moe, plain, other = layer(shared_inter=128), layer(shared_inter=128), layer(seed=6, shared_inter=128)
    plain.shared_expert = None                      # the same routed experts
    packed, gate = moe.shared_expert, moe.shared_expert_gate
    with_packed, routed = moe(x).clone(), plain(x).clone()
    calls(moe, x, with_packed)
    dense = block(1)
    moe.shared_expert = dense
    calls(moe, x, with_dense(routed, x, dense, gate))
    moe.shared_expert = packed
    calls(moe, x, with_packed)
    moe.shared_expert = other.shared_expert
    fresh = layer(shared_inter=128)
    fresh.shared_expert = other.shared_expert
    calls(moe, x, fresh(x).clone())
    moe.shared_expert_gate = None
    calls(moe, x, routed)


def test_expert_parallel_shared_expert_replaced():
    """The wrapper's own layer of the shared expert follows the expert it holds and the local module's activation mode."""
    from dartmoq_b200 import ep
    x = tokens()[0]
    a, b = layer(shared_inter=128), layer(seed=6, shared_inter=128)
    gate = a.shared_expert_gate

    def wrap(expert, cls=None):
        local = ep.shard_experts(a, 0, 8)
        if cls is not None:
            cls.from_wxa16(local)
        return ep.ExpertParallelMoE(a.gate, local, 8, 2, expert, gate)

    w = wrap(a.shared_expert)
    first = w._shared_partial(x).clone()
    w.shared_expert = b.shared_expert
    want = wrap(b.shared_expert)._shared_partial(x)
    assert not torch.equal(want, first) and torch.equal(w._shared_partial(x), want)
    w.shared_expert = block(1)
    assert w._shared_partial(x) is None             # not packed: the caller applies the module
    w.shared_expert = None
    assert w._shared_partial(x) is None
    w.shared_expert = a.shared_expert
    assert torch.equal(w._shared_partial(x), first)
    D.WxA8BitPartitionedGroupMoE.from_wxa16(w.local_moe)
    eight = wrap(a.shared_expert, D.WxA8BitPartitionedGroupMoE)._shared_partial(x)
    assert not torch.equal(eight, first) and torch.equal(w._shared_partial(x), eight)


def test_projections_of_a_packed_expert_replaced():
    """One of the packed expert's projections put in another's place, or a dense one: never the old weights."""
    from dartmoq_b200 import ep
    x = tokens()
    moe, fresh, other = layer(shared_inter=128), layer(shared_inter=128), layer(seed=6, shared_inter=128)
    wrap = ep.ExpertParallelMoE(moe.gate, ep.shard_experts(moe, 0, 8), 8, 2, moe.shared_expert, moe.shared_expert_gate)
    first, alone = moe(x).clone(), wrap._shared_partial(x[0]).clone()
    calls(moe, x, first)
    moe.shared_expert.down_proj = fresh.shared_expert.down_proj = other.shared_expert.down_proj
    want = fresh(x).clone()
    assert not torch.equal(want, first)
    calls(moe, x, want)
    again = ep.ExpertParallelMoE(moe.gate, ep.shard_experts(moe, 0, 8), 8, 2, moe.shared_expert, moe.shared_expert_gate)
    assert not torch.equal(again._shared_partial(x[0]), alone)
    assert torch.equal(wrap._shared_partial(x[0]), again._shared_partial(x[0]))
    torch.manual_seed(9)
    dense = D.W8A8Linear.from_linear(torch.nn.Linear(128, HIDDEN, bias=False, dtype=torch.bfloat16, device=DEV))
    moe.shared_expert.down_proj = dense
    plain = layer(shared_inter=128)
    plain.shared_expert = None
    routed = plain(x).clone()
    calls(moe, x, with_dense(routed, x, moe.shared_expert, moe.shared_expert_gate))
    assert wrap._shared_partial(x[0]) is None       # the caller applies the module


@pytest.mark.parametrize("assign", (False, True))
@pytest.mark.parametrize("n", (40, 700))
def test_a_state_dict_loaded_after_calls_is_used(n, assign):
    """The engine's weights are copies and captured graphs hold addresses: both are made anew after a load."""
    x, bits = tokens(n), [2, 4, 2, 4, 4, 2, 2, 4]
    a, b, c = layer(expert_bits=bits), layer(seed=6, expert_bits=bits), layer(expert_bits=bits)
    first = a(x).clone()
    calls(a, x, first)
    c.load_state_dict(b.state_dict())               # before its first call
    want = c(x).clone()
    assert not torch.equal(want, first)
    a.load_state_dict({k: v.clone() for k, v in b.state_dict().items()}, assign=assign)
    calls(a, x, want)
    for bit, w in a.bit_weights.items():
        for side in ("gate_up", "down"):
            pk = getattr(w, side + "_packed")
            assert pk["norms"] is getattr(w, side + "_norms")
    lin, other = (layer(seed=s, shared_inter=128).shared_expert.gate_proj for s in (5, 6))
    fresh = D.WxA16Linear(other.in_features, other.out_features, 8, 128, other.packed_indices, other.codebook, other.norms, lin.seed)
    lin(x[0])
    lin.load_state_dict({k: v.clone() for k, v in other.state_dict().items()}, assign=assign)
    assert torch.equal(lin(x[0]), fresh(x[0]))


@pytest.mark.parametrize("assign", (False, True))
def test_expert_parallel_weights_loaded_after_calls(assign):
    from dartmoq_b200 import ep
    x, bits = tokens()[0], [2, 4, 2, 4, 4, 2, 2, 4]
    a, b = layer(shared_inter=128, expert_bits=bits), layer(shared_inter=128, seed=6, expert_bits=bits)
    for u, v in zip(a.shared_expert.children(), b.shared_expert.children()):
        v.seed = u.seed                             # rotations are not part of a state dict

    def wrap(m):
        return ep.ExpertParallelMoE(m.gate, ep.shard_experts(m, 0, 8), 8, 2, m.shared_expert, m.shared_expert_gate)

    w, other = wrap(a), wrap(b)
    first, want = w._shared_partial(x).clone(), other._shared_partial(x).clone()
    assert not torch.equal(first, want)
    w.load_state_dict({k: v.clone() for k, v in other.state_dict().items()}, assign=assign)
    assert torch.equal(w._shared_partial(x), want)

"""Weights that modules derive from their parameters: taken anew when these change, in the memory of the old ones."""
import copy
from types import SimpleNamespace

import torch


def block(qk_norm=False):
    from rl_for_mario_b200.dt_model import DTBlock, DTConfig

    torch.manual_seed(0)
    b = DTBlock(DTConfig(hidden_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1,
                         context_len=4, qk_norm=qk_norm))
    b.fuse_norm()
    return b


def derived(b, dtype=torch.bfloat16):
    return b.self_attn._fused_weight(dtype), b.self_attn._cat_weight(dtype), b._swiglu_weight(dtype)


def test_new_weights_stand_where_the_old_ones_stood():
    b = block()
    old = derived(b)
    was = [t.clone() for t in old]
    assert all(t.grad_fn is None and not t.requires_grad for t in old)
    assert all(x is y for x, y in zip(derived(b), old))  # unchanged parameters: nothing is made
    with torch.no_grad():
        for p in b.parameters():
            p.mul_(1.5)
    new, want = derived(b), derived(copy.deepcopy(b))
    for n, o, w, x in zip(new, old, want, was):
        assert n.data_ptr() == o.data_ptr() and n.data_ptr() != w.data_ptr()
        assert torch.equal(n, w) and not torch.equal(n, x)
    # Another type is another weight.
    assert all(t.dtype == torch.float32 for t in derived(b, torch.float32))


def test_inference_mode_first():
    b = block()
    with torch.inference_mode():
        old = derived(b)
    with torch.no_grad():
        b.self_attn.k_proj.weight.add_(1.0)
        b.mlp.up_proj.weight.add_(1.0)
    new = derived(b)
    with torch.inference_mode():
        b.mlp.up_proj.weight.add_(1.0)
        again = derived(b)
    for o, n, a in zip(old, new, again):
        assert o.data_ptr() == n.data_ptr() == a.data_ptr()


def test_a_swapped_module_keeps_no_graph():
    from rl_for_mario_b200.attention import FastDTAttention

    m = FastDTAttention(SimpleNamespace(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, dropout=0.0))
    assert m._cat_weight(torch.float32).grad_fn is None
    copy.deepcopy(m)

"""The training form's checks on the host."""
import pytest
import torch


def model(**kw):
    from rl_for_mario_b200.dt_model import DTConfig, MarioDT

    cfg = DTConfig(hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, context_len=8, **kw)
    return MarioDT(cfg).train().fuse_training(seed=1)


@pytest.mark.parametrize("mask", [[0, 1, 0, 1], [1, 1, 1, 0], [0, 0, 1, 0]], ids=str)
def test_training_form_checks_masks_where_a_layer_asks_for_it(mask):
    m = model()
    data = dict(states=torch.zeros(2, 4, 4, 84, 84), actions=torch.zeros(2, 4, dtype=torch.long),
                returns_to_go=torch.zeros(2, 4), timesteps=torch.arange(4).expand(2, 4))
    bad = torch.tensor([[0, 0, 1, 1], mask])
    m.model.layers[1].self_attn.check_masks = True
    with pytest.raises(ValueError, match="left-padding"):
        m(**data, attention_mask=bad)
    # A mask that is one is taken: the refusal that follows is the kernels', of CPU tensors.
    with pytest.raises(ValueError, match="CUDA"):
        m(**data, attention_mask=torch.tensor([[0, 0, 1, 1], [0, 1, 1, 1]]))


def test_modules_pickled_before_the_training_form():
    """A module whose state holds nothing of the training form is one that is not in it."""
    m = model().model.layers[0].self_attn
    for name in ("train_form", "train_seed", "train_site", "_dropout_state"):
        m.__dict__.pop(name, None)
    with pytest.raises(ValueError, match="CUDA"):  # past the switch: the refusal is the module's own, of CPU tensors
        m(torch.zeros(1, 3, 128), (torch.zeros(3, 32), torch.zeros(3, 32)))
    assert m.train_form is False and m.train_site == 0
    assert m.dropout_state().state_dict() == {"seed": 0, "step": 0}

"""not-gpu: the types of labels and class indices, before they reach a kernel."""
import pytest
import torch

from neuron_interpolation_model_fusion_amd import ops

H, W, Z = torch.zeros(2, 8), torch.zeros(5, 8), torch.zeros(2, 5)


@pytest.mark.parametrize('dt', [torch.int8, torch.int16, torch.int32, torch.int64, torch.uint8, torch.uint16, torch.uint32, torch.uint64])
def test_indices_of_every_integer_type_keep_their_classes(dt):
    """What is too large for 32 bits is no class (its row becomes NaN), never an absent entry."""
    big = min(torch.iinfo(dt).max, 2 ** 31 - 1)
    given = torch.tensor([[0, 3, torch.iinfo(dt).max]]).to(dt) if dt != torch.uint64 else \
        torch.tensor([[0, 3, -1]]).view(torch.uint64)
    indices, _, _ = ops._top_targets(torch.zeros(1, 3), given, None)
    assert indices.dtype == torch.int32 and indices.tolist() == [[0, 3, big]]
    if dt.is_signed:
        indices, _, _ = ops._top_targets(torch.zeros(1, 2), torch.tensor([[-1, torch.iinfo(dt).min]], dtype=dt), None)
        assert (indices < 0).all()


@pytest.mark.parametrize('call', [
    lambda t: ops.linear_cross_entropy(H, W, t[:, 0]), lambda t: ops.linear_topk_distillation(H, W, torch.zeros(2, 3), t),
    lambda t: ops.topk_distillation(Z, torch.zeros(2, 3), t)])
@pytest.mark.parametrize('dt', [torch.float32, torch.bool, torch.complex64])
def test_other_types_are_refused(call, dt):
    with pytest.raises((TypeError, ValueError), match='integers'):
        call(torch.zeros(2, 3, dtype=dt))


def _wide(*shape):
    return torch.zeros(1).expand(*shape)  # no memory behind it


@pytest.mark.parametrize('call', [
    lambda: ops.linear_cross_entropy(_wide(2, 1), _wide(2 ** 32 + 5, 1), torch.zeros(2, dtype=torch.int64)),
    lambda: ops.linear_cross_entropy(_wide(2, 2 ** 32 + 8), _wide(5, 2 ** 32 + 8), torch.zeros(2, dtype=torch.int64)),
    lambda: ops.linear_cross_entropy(_wide(2 ** 31, 8), W, torch.zeros(1, dtype=torch.int64).expand(2 ** 31)),
    lambda: ops.linear_cross_entropy(_wide(2 ** 29, 8), _wide(2 ** 15, 8), torch.zeros(1, dtype=torch.int64).expand(2 ** 29)),
    lambda: ops.linear_topk_distillation(_wide(2, 1), _wide(2 ** 28 + 1, 1), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)),
    lambda: ops.topk_distillation(_wide(2, 2 ** 32 + 5), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32)),
    lambda: ops.topk_distillation(_wide(2 ** 31, 5), _wide(2 ** 31, 3), torch.zeros(1, dtype=torch.int32).expand(2 ** 31, 3)),
    lambda: ops.top_logits(_wide(2, 2 ** 32 + 5), 3),
    lambda: ops.top_logits(_wide(3, 2 ** 31, 5), 3)])
def test_sizes_beyond_the_limits_are_refused(call):
    """Not cut to 32 bits: 2^32 + 5 classes are not 5."""
    with pytest.raises(ValueError, match='at most'):
        call()

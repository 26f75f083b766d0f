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

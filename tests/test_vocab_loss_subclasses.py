"""Tensors whose storage does not hold their values, which the losses' kernels would
take for none: the entry points refuse them."""
import pytest
import torch

from moc_amd import losses as L


class Wrapper(torch.Tensor):
    """Holds another tensor; its own storage is empty."""

    @staticmethod
    def __new__(cls, held):
        return torch.Tensor._make_wrapper_subclass(cls, held.shape, dtype=held.dtype, device=held.device)

    def __init__(self, held):
        self.held = held

    @classmethod
    def __torch_dispatch__(cls, func, types, args, kwargs):
        return cls(func(*[a.held if isinstance(a, Wrapper) else a for a in args], **(kwargs or {})))


INPUTS = dict(hidden=torch.zeros(6, 8), weight=torch.zeros(10, 8), logits=torch.zeros(6, 10),
              labels=torch.zeros(6, dtype=torch.int64), teacher_ids=torch.zeros(6, 4, dtype=torch.int32),
              teacher_logits=torch.zeros(6, 4), row_weight=torch.ones(6))
TAKES = {"linear_cross_entropy": ("hidden", "weight", "labels", "row_weight"),
         "linear_distillation": ("hidden", "weight", "teacher_ids", "teacher_logits", "row_weight"),
         "distillation_loss": ("logits", "teacher_ids", "teacher_logits", "row_weight")}


@pytest.mark.parametrize("name,wrapped", [(name, arg) for name, args in TAKES.items() for arg in args])
def test_refused(name, wrapped):
    assert Wrapper(INPUTS["row_weight"]).reshape(6).contiguous().data_ptr() == 0
    args = {arg: Wrapper(INPUTS[arg]) if arg == wrapped else INPUTS[arg] for arg in TAKES[name]}
    with pytest.raises(ValueError, match="plain tensors only"):
        getattr(L, name)(**args)

"""TopLogitsDistillLoss takes the same lists on the host as on the device, and answers alike: types, shapes, gradients."""
import pytest
import torch

from ponderv2_amd.ponder.models.losses import LOSSES
from row_ops_oracle import EPS32, distill, half_step
from test_distill_loss import lists


@pytest.fixture(params=["host", pytest.param("device", marks=pytest.mark.gpu)])
def where(request):
    return request.getfixturevalue("device") if request.param == "device" else torch.device("cpu")


def criterion(**options):
    return LOSSES.build(cfg=dict(type="TopLogitsDistillLoss", **options))


def test_refusals_are_the_same(where):
    index, teacher = (t.to(where) for t in lists(8, 9, 3))
    for pred in (torch.randn(8, 9, device=where), torch.randn(8, 9, device=where, dtype=torch.float64)):
        for bad in (index.float(), index.short(), index.bool()):
            with pytest.raises(TypeError, match="int64 or int32"):
                criterion()(pred, (bad, teacher))
        for bad in (teacher.double(), teacher.long()):
            with pytest.raises(TypeError, match="teacher_logits expected"):
                criterion()(pred, (index, bad))
        for bad in ((index[:7], teacher[:7]), (index[:, :2], teacher), (index[0], teacher[0]), (index[:1], teacher[:1])):
            with pytest.raises(ValueError, match="expected, got"):
                criterion()(pred, bad)
        with pytest.raises(ValueError, match="0 listed"):
            criterion()(pred, (index[:, :0], teacher[:, :0]))
        with pytest.raises(ValueError, match="1025 listed"):
            criterion()(pred, (index[:, :1].expand(8, 1025), teacher[:, :1].expand(8, 1025)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_types_and_gradients_are_the_same(where, dtype):
    """fp32 (fp64 of fp64 logits) whatever the logits' type, gradients in the logits' type and of the logits only."""
    torch.manual_seed(30)
    index, teacher = (t.to(where) for t in lists(40, 17, 5))
    pred = (torch.randn(40, 17, device=where) * 2).to(dtype).requires_grad_()
    teacher.requires_grad_()
    for some in (index, index.int()):
        loss = criterion(temperature=2.0, reduction="sum")(pred, (some, teacher))
        assert loss.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
        grad, none = torch.autograd.grad(loss, (pred, teacher), allow_unused=True)
        assert none is None and grad.dtype == dtype
        rows, want, _, big, *_ = distill(pred.detach(), index, teacher.detach(), 2.0)
        # a row: T^2 (8 |log| + 48) (2 + 2 |log|) roundings of fp32; 40 rows and their sum
        row = 4 * (8 * float(big.max()) + 48) * (2 + 2 * float(big.max())) * EPS32
        assert abs(float(loss.detach()) - float(rows.sum())) <= 40 * row + 64 * EPS32 * float(rows.sum())
        bound = want.abs() * half_step(dtype) * 1.01 + 2 * (8 * float(big.max()) + 64) * EPS32 + 2.0 ** -24
        assert bool(((grad.double() - want).abs() <= bound).all())

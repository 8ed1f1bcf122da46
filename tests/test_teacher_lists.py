"""A teacher's lists (teacher_index, teacher_logits) stay with their points through every transform that selects or reorders
points, on the host and in the device half of the grid sampling.  Each list holds its own point's number."""
import numpy as np
import pytest
import torch

from ponderv2_amd.ponder.datasets.collate import point_collate_fn
from ponderv2_amd.ponder.datasets.transform import Compose
from ponderv2_amd.ponder.datasets.voxelize import device_grid_sample
from ponderv2_amd.ponder.models.losses import build_criteria
from ponderv2_amd.ponder.models.ponder.ponder_indoor_base import PonderIndoor
from test_distill_loss import ppt

N, K = 3000, 4


def sample(seed):
    """Points whose coordinates, labels and lists tell which point they are of."""
    rng = np.random.RandomState(seed)
    number = np.arange(N)
    coord = rng.uniform(0, 1, (N, 3))
    return dict(coord=coord, color=rng.rand(N, 3), normal=rng.rand(N, 3), strength=number[:, None] / N,
                segment=number.copy(), instance=number.copy(),
                teacher_index=number[:, None] * 10 + np.arange(K),
                teacher_logits=(number[:, None] + np.arange(K) / 10).astype(np.float32))


def check(data, fewer=True):
    number = np.asarray(data["segment"])
    assert (len(number) < N) == fewer and len(np.unique(number)) == len(number)
    assert np.array_equal(np.asarray(data["teacher_index"]), number[:, None] * 10 + np.arange(K))
    assert np.array_equal(np.asarray(data["teacher_logits"]), (number[:, None] + np.arange(K) / 10).astype(np.float32))


TRANSFORMS = {
    "dropout": dict(type="RandomDropout", dropout_ratio=0.5, dropout_application_ratio=1.0),
    "shuffle": dict(type="ShufflePoint"),
    "range": dict(type="PointRangeFilter", point_cloud_range=(0, 0, 0, 0.8, 0.9, 1.0)),
    "grid": dict(type="GridSample", grid_size=0.1),
    "grid, named": dict(type="GridSample", grid_size=0.1, keys=("coord", "segment", "teacher_logits")),
}


@pytest.mark.parametrize("name", TRANSFORMS)
def test_one_transform(name):
    np.random.seed(0)
    check(Compose([TRANSFORMS[name]])(sample(1)), fewer=name != "shuffle")


def test_labelled_points_stay_with_their_lists():
    np.random.seed(1)
    data = sample(2)
    data["sampled_index"] = np.arange(0, N, 17)
    out = Compose([TRANSFORMS["dropout"]])(data)
    check(out)
    assert set(range(0, N, 17)) <= set(out["segment"].tolist())


def chain(*more):
    return Compose([TRANSFORMS["dropout"], TRANSFORMS["range"], *more, dict(type="ShufflePoint"), dict(type="ToTensor"),
                    dict(type="Collect", keys=("coord", "segment", "teacher_index", "teacher_logits"),
                         feat_keys=("color", "normal"))])


def test_a_chain():
    np.random.seed(2)
    out = chain(TRANSFORMS["grid"])(sample(3))
    check(out)
    assert out["teacher_index"].dtype == torch.int64 and out["teacher_logits"].dtype == torch.float32


def test_grid_sampling_of_a_batch():
    """The trainer's device half: raw points of several scenes, one representative per voxel."""
    np.random.seed(3)
    batch = point_collate_fn([chain()(sample(4)), chain()(sample(5))])
    for keys in (("coord", "feat", "segment"), ("coord", "segment", "teacher_index")):
        out = device_grid_sample(batch, grid_size=0.1, keys=keys)
        ends = [0, *out["offset"].tolist()]
        assert ends[-1] == len(out["coord"]) < len(batch["coord"])
        for a, b in zip(ends[:-1], ends[1:]):
            check({k: out[k][a:b] for k in ("segment", "teacher_index", "teacher_logits")})


def test_samples_without_lists_are_as_before():
    np.random.seed(4)
    data = sample(6)
    del data["teacher_index"], data["teacher_logits"]
    with_lists, without = sample(6), data
    for transforms in (list(TRANSFORMS.values())[:4],):
        np.random.seed(5)
        a = Compose(transforms)(with_lists)
        np.random.seed(5)
        b = Compose(transforms)(without)
        assert "teacher_index" not in b
        for k in b:
            assert np.array_equal(a[k], b[k]), k


@pytest.mark.parametrize("missing", [("teacher_index", "teacher_logits"), ("teacher_logits",), ("teacher_index",)])
def test_a_batch_without_lists_is_refused_by_name(missing):
    """As a dataset without a teacher among others brings it; the other criteria do not ask for lists."""
    model, batch = ppt(torch.device("cpu"))
    for key in missing:
        del batch[key]
    with pytest.raises(ValueError, match="TopLogitsDistillLoss: the batch carries no teacher's lists"):
        PonderIndoor.ppt_loss(model, batch)
    model.ppt_criteria = build_criteria([dict(type="CrossEntropyLoss", loss_weight=1.0, ignore_index=-1)])
    assert torch.isfinite(PonderIndoor.ppt_loss(model, batch))


def test_criteria_of_two_arguments():
    """A model whose criteria are a callable (pred, target) of its own is called with two, as ever, lists in the batch or not."""
    model, batch = ppt(torch.device("cpu"))
    model.ppt_criteria = lambda pred, target: torch.nn.functional.cross_entropy(pred, target, ignore_index=-1)
    assert torch.isfinite(PonderIndoor.ppt_loss(model, batch))
    del batch["teacher_index"], batch["teacher_logits"]
    assert torch.isfinite(PonderIndoor.ppt_loss(model, batch))

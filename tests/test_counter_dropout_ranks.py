"""Counter dropout in data-parallel training: every rank draws masks of its own, from the same weights."""
import pytest
import torch

from dist_util import run_ranks
from xnn_b200.data import AtomicDataset, synthetic
from xnn_b200.ops import CounterDropout, counter_dropout


def _rank(rank, world, out_dir, seeds):
    from xnn_b200.config import from_dict
    from xnn_b200.train import Trainer
    cfg = from_dict({"model": {"name": "schnet", "cutoff": 4.0, "n_features": 8, "n_interactions": 1, "n_rbf": 6},
                     "optim": {"epochs": 1, "force_weight": 0.0}, "data": {"batch_size": 2, "val_fraction": 0.0},
                     "trainer": {"loggers": []}, "device": "cpu", "seed": 3, "output_dir": str(out_dir)})
    torch.manual_seed(10 + rank if seeds else 3)
    from xnn_b200.models import prepare_model
    model = prepare_model(cfg)
    model.drop = CounterDropout(0.5, seed=seeds[rank] if seeds else None)
    model.register_buffer("count", torch.tensor([float(rank)]))
    tr = Trainer(cfg, AtomicDataset(synthetic.small_organic(4, seed=1), 4.0), val=[], test=[], model=model)
    x = torch.ones(4096)
    masks = [model.drop(x) != 0 for _ in range(3)]
    out = {"masks": torch.stack(masks), "seed": int(model.drop.rng[0]), "count": float(model.count),
           "weights": torch.cat([p.detach().reshape(-1) for p in tr.module.parameters()])}
    tr.close()
    return out


@pytest.mark.parametrize("seeds", [None, (7, 8)])
def test_ranks_draw_different_masks(tmp_path, seeds):
    a, b = run_ranks(_rank, 2, str(tmp_path), seeds)
    assert torch.equal(a["weights"], b["weights"]) and a["count"] == b["count"] == 0.0
    assert [a["seed"], b["seed"]] == (list(seeds) if seeds else [a["seed"]] * 2)
    for x in a["masks"]:
        for y in b["masks"]:
            # independent halves: of 4096 entries 2048 agree, with a standard deviation of 32
            assert abs(int((x == y).sum()) - 2048) < 6 * 32
    # rank 0 draws what a single process draws
    one = CounterDropout(0.5, seed=a["seed"])
    assert all(torch.equal(one(torch.ones(4096)) != 0, m) for m in a["masks"])


def test_rank_sets_where_the_offset_counts_from():
    drop, x = CounterDropout(0.5, seed=9), torch.ones(512)
    drop(x)
    for rank in (0, 3, 3):
        drop.set_rank(rank)
        at = int(drop.rng[1])
        assert at >> 40 == rank
        assert torch.equal(drop(x), counter_dropout(x, 0.5, (9, at))) and int(drop.rng[1]) == at + 1

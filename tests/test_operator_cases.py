"""The inputs of the served operators' performance cases are determined by the seed alone."""
import random

import pytest
import torch

from perf import operators


def sampling_cases():
    rng = random.Random(1)
    drawn = [operators.draw(rng) for _ in range(60)]
    small = [c for c in drawn if c["op"] == "sample" and c["rows"] * c["vocab"] < 3e6]
    return [c for c in operators.listed() if c["op"] == "sample" and c["rows"] * c["vocab"] < 4e6] + small[:4]


@pytest.mark.parametrize("case", sampling_cases(), ids=lambda c: f"{c['rows']}x{c['vocab']}")
def test_no_logit_is_written_twice(monkeypatch, case):
    """Where one call writes a place twice, which of the values stays is not determined on a GPU."""
    monkeypatch.setattr(operators, "DEVICE", "cpu")
    scatter, seen = torch.Tensor.scatter_, []

    def recorded(self, dim, index, *args):
        seen.append((self.shape, dim, index))
        return scatter(self, dim, index, *args)
    monkeypatch.setattr(torch.Tensor, "scatter_", recorded)
    for seed in (1, 2, 3):
        operators.prepare(case, seed)
    assert seen
    for shape, dim, index in seen:
        ordered = index.sort(dim).values
        assert bool((ordered.diff(dim=dim) > 0).all())
        assert int(index.min()) >= 0 and int(index.max()) < shape[dim]

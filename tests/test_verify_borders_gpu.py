"""Sampled verification (paged.verify_picks) where a temperature is small against the
spacing of the logits, and where much of a sum is taken off: equal picks with the
definition in 64 bits (q4_ref.verify), whose decisions are asserted to be clear."""
import numpy as np
import pytest
import torch

from tests import q4_ref
from tests.test_verify_gpu import make, run, wanted

pytestmark = pytest.mark.gpu


def below(top, n):
    """top and the n - 1 floats under it, in order."""
    x = [np.float32(top)]
    while len(x) < n:
        x.append(np.nextafter(x[-1], np.float32(-np.inf), dtype=np.float32))
    return np.array(x, np.float32)


def cold_case(many):
    """Rows that hold the floats under their largest (twice the largest), with
    temperatures at which e^-690, the least weight that counts, lies among them; a root
    with two children, of which the first has next to no weight and the second half."""
    V = 96
    rows, heat = [], []
    for top in (20.0, 1500.0, 0.1, 3.0e-24, -7.0, 1.0e30):
        x = below(top, V - 1)
        gap = float(x[0]) - float(x[1])
        for at in (0.3, 0.5, 0.6, 0.7, 0.9, 1.0, 1.3, 1.5, 2.0, 2.5, 4.0, 6.0, 6.5, 20.0):
            rows.append(np.concatenate([x[:1], x]))
            heat.append(gap * at / 690)
    rows, heat = rows[:many], heat[:many]
    n = len(rows)
    rng = np.random.default_rng(4)
    x = np.zeros((3 * n, V), np.float32)
    tokens = np.zeros(3 * n, np.int64)
    for b in range(n):
        place = rng.permutation(V)  # where each of them stands
        x[3 * b, place] = rows[b]
        x[3 * b + 1:3 * b + 3, b % V] = 1.0
        tokens[3 * b + 1] = place[2 + b % 5]  # one to five floats under the largest
        tokens[3 * b + 2] = place[b % 2]
    u = np.tile(np.array([0, 0.3, 0.0], np.float32), n)
    u[2::3] = np.where(np.arange(n) % 3 == 0, 0.2, 0.9)  # taken, and turned down
    return dict(x=x, cu=(3 * np.arange(n + 1)).tolist(), parents=[-1, 0, 0] * n, tokens=tokens, u=u,
                d=(0.2603 + 0.4808 * (np.arange(n) % 2)).astype(np.float32), T=np.array(heat, np.float32), q=None)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("many", [12, 84])  # a cluster per node, and per request
def test_temperatures_small_against_the_logits_spacing(cuda_dev, many, draft):
    c = cold_case(many)
    assert (c["T"] > 0).all()
    if draft:
        c["q"] = np.full(c["x"].shape, 1.0 / c["x"].shape[1], np.float32)
    picks, margin, drawn = q4_ref.verify(c["x"], c["cu"], c["parents"], c["tokens"], c["u"], c["d"], c["T"], c["q"])
    assert margin > 2e-5 and drawn > 1e-11
    got = run(cuda_dev, c, "f32", max_nodes=3)
    assert np.array_equal(got, picks), np.nonzero(got != picks)[0]


@pytest.mark.parametrize("dt,singles", [("f32", 0), ("f16", 0), ("f16", 36)])
@pytest.mark.parametrize("side", [-1, 1])
def test_what_is_left_of_a_long_sum(cuda_dev, dt, singles, side):
    """Two million like weights behind one that has 10 of 11 parts of the sum and is turned
    down; the next child's number lies 1e-4 of itself beside its share of what is left.
    A sum of weights e^-y is off by at most 2^-22 (7 + y) of each: for the large one, ten
    times what is left, 1.7e-5 of that, for the others (y = 17) 5.8e-6."""
    V = 2000000
    at = 123456
    ratio = 0.3 / 1.3
    n = 3 + singles
    x = np.zeros((n, V), np.float32)
    x[0, at] = np.log(0.3 * V)
    x[0, 0] = np.log(10 * 1.3 * V)
    x = torch.from_numpy(x).to(torch.float16 if dt == "f16" else torch.float32).float().numpy()
    big, second = np.exp(x[0, [0, at]].astype(np.float64))
    left = second + V - 2
    u = np.zeros(n, np.float32)
    u[1] = 0.99
    u[2] = second / left * (1 + side * 1e-4)
    assert abs(second / left - ratio) < 0.01 and left / (left + big) > 1 / 16  # not summed up anew
    tokens = np.zeros(n, np.int64)
    tokens[2] = at
    rng = np.random.default_rng(8)
    c = dict(x=x, cu=[0] + list(range(3, n + 1)), parents=[-1, 0, 0] + [-1] * singles, tokens=tokens, u=u,
             d=rng.random(1 + singles).astype(np.float32), T=None, q=None)
    picks, margin, drawn = q4_ref.verify(x, c["cu"], c["parents"], tokens, u, c["d"], None, None)
    assert margin > 9e-5 and drawn > 1e-11 and (picks[0] == at) == (side < 0)
    assert np.array_equal(run(cuda_dev, c, dt, max_nodes=3), picks)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("nodes", [[6], [20, 30, 4], [3] * 50])
def test_stars_with_high_numbers(cuda_dev, draft, nodes):
    """Children of a root, likely tokens, nearly all turned down: four cases whose
    decisions are clear."""
    seen = 0
    for seed in range(200):
        c = make(nodes, 400, "f32", draft, "star", np.random.default_rng(seed), agree=1.0)
        c["u"] = np.maximum(c["u"], np.float32(0.9))
        picks, margin, drawn = wanted(c)
        if margin > 2e-5 and drawn > 1e-11:
            assert np.array_equal(run(cuda_dev, c, "f32"), picks)
            seen += 1
            if seen == 4:
                return
    raise AssertionError(f"{seen} clear cases")

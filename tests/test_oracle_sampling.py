"""The sampling oracle against its definition by cases and by frequency (CPU)."""
import numpy as np

from oracle.sampling import sample_f64


def test_known_rows():
    z = np.log([0.1, 0.4, 0.2, 0.3])
    assert [sample_f64(z, u)[0] for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [sample_f64(z, u, top_k=2)[0] for u in (0.0, 0.57, 0.58)] == [1, 1, 3]
    # 0.4 before the second, 0.7 before the third: 0.6 keeps two tokens, 0.71 three
    assert {sample_f64(z, u, top_p=0.6)[0] for u in np.linspace(0, 0.999, 50)} == {1, 3}
    assert {sample_f64(z, u, top_p=0.71)[0] for u in np.linspace(0, 0.999, 50)} == {1, 2, 3}
    assert {sample_f64(z, u, top_p=0.0)[0] for u in np.linspace(0, 0.999, 50)} == {1}
    # 0.3 / 0.4 = 0.75
    assert {sample_f64(z, u, min_p=0.74)[0] for u in np.linspace(0, 0.999, 50)} == {1, 3}
    assert sample_f64(z, 0.999, temperature=0.0)[0] == 1
    # top-p counts among what top-k leaves: of {0.4, 0.3} a share of 0.6 needs both
    assert {sample_f64(z, u, top_k=2, top_p=0.6)[0] for u in np.linspace(0, 0.999, 50)} == {1, 3}
    assert {sample_f64(z, u, top_k=2, top_p=0.55)[0] for u in np.linspace(0, 0.999, 50)} == {1}


def test_ties_and_empty_rows():
    z = np.zeros(8)
    assert [sample_f64(z, u)[0] for u in (0.0, 0.125, 0.4999, 0.5)] == [0, 1, 3, 4]
    assert {sample_f64(z, u, top_k=3)[0] for u in np.linspace(0, 0.999, 50)} == {0, 1, 2}
    assert {sample_f64(z, u, top_p=0.5)[0] for u in np.linspace(0, 0.999, 50)} == {0, 1, 2, 3}
    assert sample_f64(np.full(4, -np.inf), 0.5)[0] == -1
    assert sample_f64(np.array([np.nan, -np.inf, 1.0]), 0.9)[0] == 2
    assert {sample_f64(np.array([1.0, np.inf, 0.0, np.inf]), u)[0] for u in (0.0, 0.4, 0.6)} == {1, 3}


def test_frequencies():
    rng = np.random.default_rng(0)
    z = rng.standard_normal(12) * 2
    p = np.exp(z / 0.8)
    n = 20000
    got = np.bincount([sample_f64(z, (i + 0.5) / n, temperature=0.8)[0] for i in range(n)], minlength=12) / n
    assert np.abs(got - p / p.sum()).max() <= 1.0 / n

"""The example's model: its gradients through every operator against differences, its training, its answers."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("window_language_model", os.path.join(ROOT, "examples", "window_language_model.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def batch(example, D, window):
    alphabet = sorted(set(example.TEXT))
    tokens = np.array([alphabet.index(c) for c in example.TEXT])
    windows, follows = example.windows_of(tokens, window)
    return len(alphabet), windows, follows


@pytest.mark.parametrize("bonus", [0.0, 0.3])
def test_gradients_against_differences(gpu, D, example, bonus):
    vocab, windows, follows = batch(example, D, 3)
    model = example.WindowModel(vocab, window=3, embedding=5, hidden=17, dtype=np.float64, seed=3)
    w, f = D.Array.from_numpy(windows[:60]), D.Array.from_numpy(follows[:60])
    _, gradients = model.loss_and_gradients(w, f, bonus)
    gradients = [g.numpy() for g in gradients]
    rng, step = np.random.RandomState(1), 1e-5
    for name, gradient in zip(model.NAMES, gradients):
        value = getattr(model, name).numpy()
        along = rng.randn(*value.shape)
        ends = []
        for sign in (1, -1):
            setattr(model, name, D.Array.from_numpy(value + sign * step * along))
            ends.append(float(model.loss_and_gradients(w, f, bonus)[0].numpy()))
        setattr(model, name, D.Array.from_numpy(value))
        # the loss is of order one and its third derivative along `along` of order |along|^3 (a few hundred at most), its rounding some 1e-15 a difference
        assert abs((ends[0] - ends[1]) / (2 * step) - (gradient * along).sum()) <= np.linalg.norm(along) ** 3 * step ** 2 * 10 + 1e-14 / step, name


def test_training_and_answers(gpu, D, example):
    vocab, windows, follows = batch(example, D, 6)
    model = example.WindowModel(vocab)
    w, f = D.Array.from_numpy(windows), D.Array.from_numpy(follows)
    losses = []
    for _ in range(120):
        loss, norm = model.step(w, f, rate=0.5)
        losses.append(float(loss.numpy()))
        assert np.isfinite(norm.numpy())
    # from about the logarithm of the vocabulary to less than half of it
    assert losses[0] > 0.8 * np.log(vocab) and losses[-1] < 0.5 * np.log(vocab)
    said = model.answer(windows[0], 5, k=4)
    assert len(said) == 5
    for alternatives in said:
        values = [p for _, p in alternatives]
        assert len(alternatives) == 4 and values == sorted(values, reverse=True) and np.exp(values).sum() <= 1 + 1e-6


def test_the_norm_of_the_step_is_bounded(gpu, D, example):
    vocab, windows, follows = batch(example, D, 6)
    model = example.WindowModel(vocab, seed=9)
    before = [p.numpy() for p in model.parameters()]
    _, norm = model.step(D.Array.from_numpy(windows), D.Array.from_numpy(follows), rate=1.0, max_norm=0.01)
    moved = np.sqrt(sum(((p.numpy().astype(np.float64) - b) ** 2).sum() for p, b in zip(model.parameters(), before)))
    # (a parameter of size one is rounded to 2^-24 when it moves; there are some 10^4)
    assert float(norm.numpy()) > 0.01 and abs(moved - 0.01) <= 1e-4

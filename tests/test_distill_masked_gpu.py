"""Distillation from rows whose masked classes have logits of -inf: rows that are held in registers (up to
65536 classes) and rows that are read twice have one meaning. Bounds: tests/token_oracle.py."""
import numpy as np
import pytest

from tests.test_token_steps_gpu import check_distill, floats

pytestmark = pytest.mark.gpu
WIDTHS = [3000, 65533, 65536, 65537, 70000, 100001, 131072]


def masked_rows(rng, C):
    """Rows with classes masked in front, in the middle, in turn, and all but one; and the classes left."""
    c = np.arange(C)
    masks = [c < 4, c < 16, c < C // 2, c < min(4096, C - 9), c < min(8192, C - 9), (c >= 4) & (c < min(4096, C - 9)),
             (c >= 1000) & (c < 1008), (c >= 2801) & (c < 2812), c // 4096 % 2 == 0 if C > 4096 else c // 64 % 2 == 0,
             c // 8 % 2 == 0, c != C - 5, c != 0, c >= 9, c >= C - 100]
    z = (floats(rng, len(masks), C) * 4).astype(np.float32)
    for row, mask in zip(z, masks):
        row[mask] = -np.inf
    return z, [c[~mask] for mask in masks]


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("grad", [True, False])
def test_masked_classes(ctx, C, grad):
    rng = np.random.default_rng(C)
    z, left = masked_rows(rng, C)
    K = 7
    index, t = np.full((len(z), K), -1), floats(rng, len(z), K) * 3
    for r, classes in enumerate(left):
        n = min(K, len(classes))
        index[r, :n] = rng.permutation(classes)[:n]
    for r in range(len(z)):  # each by itself, so that a row names itself
        check_distill(ctx, z[r:r + 1], index[r:r + 1], t[r:r + 1], grad=grad)
    # beside each other: rows of odd widths begin at every place of a group of four
    check_distill(ctx, z, index, t, 2.0, -0.5, "i64", grad)


@pytest.mark.parametrize("C", WIDTHS)
def test_a_row_without_any_class_left(ctx, C):
    """0 / 0: NaN throughout."""
    check_distill(ctx, np.full((1, C), -np.inf, np.float32), np.array([[0, C - 1]]), np.ones((1, 2), np.float32))


@pytest.mark.parametrize("C", [1, 2, 3, 4, 5])
def test_narrow_rows_with_one_class_left(ctx, C):
    rng = np.random.default_rng(C)
    z = np.full((9, C), -np.inf, np.float32)
    keep = rng.integers(0, C, 9)
    z[np.arange(9), keep] = floats(rng, 9) * 3
    check_distill(ctx, z, keep[:, None], floats(rng, 9, 1))


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("where", ["first", "last", "every"])
def test_nan_beside_masked_classes(ctx, C, where):
    """A row with a NaN is NaN throughout, also where a thread's other classes are all masked: eight
    classes of every 4096 hold a whole group of four of one thread, however the row is aligned."""
    rng = np.random.default_rng(C)
    z = (floats(rng, 3, C) * 4).astype(np.float32)
    blocks = np.arange(20, C - 8, 4096)
    nan = {"first": blocks[:1], "last": blocks[-1:], "every": blocks}[where]
    for b in blocks:
        z[:, b:b + 8] = -np.inf
    for b in nan:
        z[:, b:b + 8] = np.nan
    for r in range(3):
        check_distill(ctx, z[r:r + 1], np.array([[1, 2, 3]]), np.ones((1, 3), np.float32))
    check_distill(ctx, z, np.tile([1, 2, 3], (3, 1)), np.ones((3, 3), np.float32))

"""Minimax polynomial of 2^f on [-1/2, 1/2] for the paged attention's weights.

Remez exchange on the relative error p(f) / 2^f - 1: solve for the coefficients
that make the error alternate with equal size at n + 2 points, move the points
to the extrema, repeat. Prints the coefficients (f32) of degree n, lowest
first, and the largest relative error of the rounded polynomial.
"""
import sys

import numpy as np


def fit(n: int) -> tuple[np.ndarray, float]:
    x = np.sort(np.cos(np.pi * (np.arange(n + 2) + 0.5) / (n + 2)) * 0.5)
    grid = np.linspace(-0.5, 0.5, 200001)
    for _ in range(50):
        a = np.empty((n + 2, n + 2))
        a[:, : n + 1] = x[:, None] ** np.arange(n + 1) / 2.0 ** x[:, None]
        a[:, n + 1] = (-1.0) ** np.arange(n + 2)
        c = np.linalg.solve(a, np.ones(n + 2))[:-1]
        err = np.polynomial.polynomial.polyval(grid, c) / 2.0 ** grid - 1.0
        turns = np.flatnonzero(np.diff(np.sign(np.diff(err)))) + 1
        at = np.concatenate([[0], turns, [grid.size - 1]])
        keep = [at[0]]
        for i in at[1:]:
            if err[i] * err[keep[-1]] > 0:
                keep[-1] = max(keep[-1], i, key=lambda j: abs(err[j]))
            else:
                keep.append(i)
        if len(keep) < n + 2:
            break
        x = grid[keep[: n + 2]]
    c32 = c.astype(np.float32)
    return c32, float(np.abs(np.polynomial.polynomial.polyval(grid, c32.astype(float)) / 2.0 ** grid - 1.0).max())


if __name__ == "__main__":
    coef, worst = fit(int(sys.argv[1]) if len(sys.argv) > 1 else 4)
    print(", ".join(float(v).hex() for v in coef), "worst relative error", worst)

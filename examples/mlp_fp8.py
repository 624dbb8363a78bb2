"""An MLP trained and served in 8 bits, beside the same program in f32.

    python examples/mlp_fp8.py [--rows 4096] [--steps 200]

Two hidden layers (sigmoid, tanh) on a synthetic regression, full-batch gradient descent
through the tape.  Both programs start from the same weights.  The 8-bit one multiplies
e4m3 codes, keeps one byte an activation for its backward pass, and answers single rows
from weights held in 8 bits.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import cleave_amd as ca  # noqa: E402
from cleave_amd import autograd as ad  # noqa: E402

LAYERS = (784, 500, 300, 10)


def forward_f32(x, w):
    return ad.tanh(ad.sigmoid(x @ w[0]) @ w[1]) @ w[2]


def forward_fp8(x, w):
    h = ad.sigmoid_fp8(ad.linear_fp8(x, w[0], dtype="bf16"))
    h = ad.tanh_fp8(ad.linear_fp8(h, w[1], dtype="bf16"))
    return ad.linear_fp8(h, w[2])


def train(forward, x, y, weights, steps: int, lr: float):
    """The loss of each step, and the trained weights."""
    w = [ca.from_numpy(a) for a in weights]
    data, target, losses = ad.const(x), ad.const(y), []
    for _ in range(steps):
        p = [ad.param(t) for t in w]
        e = forward(data, p) - target
        loss = ad.mean(e * e)
        ad.backward(loss)
        for v in p:
            ca.sgd_update(v.tensor, v.grad, lr)
        losses.append(float(loss.numpy()[0]))
    return losses, w


def held(w):
    """The weights as a server keeps them: in 8 bits, N x K, so that a row's product reads each once."""
    return [ca.quantize_fp8(ca.from_numpy(np.ascontiguousarray(t.numpy().T)), block_rows=128) for t in w]


def answer(w8, rows: np.ndarray) -> np.ndarray:
    h, _ = ca.sigmoid_fp8(ca.linear_fp8(ca.from_numpy(rows), w8[0], trans_b=True), save=False)
    h, _ = ca.tanh_fp8(ca.matmul_fp8(h, w8[1], trans_b=True), save=False)
    return ca.matmul_fp8(h, w8[2], trans_b=True).numpy()


def main(rows: int = 4096, steps: int = 200, lr: float = 0.05) -> dict:
    if rows < 1 or steps < 1:
        raise ValueError(f"at least one row and one step, not {rows} and {steps}")
    rng = np.random.default_rng(7)
    x = rng.standard_normal((rows, LAYERS[0]), np.float32)
    shape = list(zip(LAYERS[:-1], LAYERS[1:]))
    teacher = rng.standard_normal((LAYERS[0], LAYERS[-1]), np.float32) / np.float32(np.sqrt(LAYERS[0]))
    y = np.tanh(x @ teacher)
    weights = [(rng.standard_normal(s, np.float32) / np.float32(np.sqrt(s[0]))) for s in shape]
    f32, _ = train(forward_f32, x, y, weights, steps, lr)
    fp8, w = train(forward_fp8, x, y, weights, steps, lr)
    w8 = held(w)
    answers = np.concatenate([answer(w8, x[i:i + 1]) for i in range(min(8, rows))])
    return {"loss_f32": f32, "loss_fp8": fp8, "served_error": float(np.abs(answers - y[:8]).mean()),
            "answers": answers, "weights": w, "x": x}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=200)
    a = ap.parse_args()
    r = main(a.rows, a.steps)
    for i in range(0, a.steps, max(1, a.steps // 8)):
        print(f"step {i:4d}  loss  f32 {r['loss_f32'][i]:.5f}   8-bit {r['loss_fp8'][i]:.5f}")
    print(f"last       loss  f32 {r['loss_f32'][-1]:.5f}   8-bit {r['loss_fp8'][-1]:.5f}")
    print(f"single rows served in 8 bits: mean |error| {r['served_error']:.4f}")

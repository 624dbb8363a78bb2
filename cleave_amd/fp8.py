"""Dense layers in 8 bits: matrices as e4m3 codes with a power-of-two scale for each block
of 128, their products, and activations kept in 8 bits for the backward pass.

    quantize_fp8(x), dequantize_fp8(t)        by rows (1 x 128 blocks), or by 128 x 128 for a weight
    matmul_fp8(a, b)                          a b or a b^T of two held matrices
    linear_fp8(x, w, x8=...)                  quantise x, multiply, keep the quantised x
    weight_grad_fp8(x8, g)                    x^T g from the kept input
    relu_fp8 / sigmoid_fp8 / tanh_fp8         act(z) in 8 bits, and z kept for ...
    relu_bwd_fp8 / sigmoid_bwd_fp8 / tanh_bwd_fp8   ... dz = g act'(z)

A layer y = x w and its gradients, forward and back:

    w8 = quantize_fp8(w, block_rows=128)           # after each update
    x8 = empty_fp8(x.shape)
    z = linear_fp8(x, w8, x8=x8)
    h8, z8 = sigmoid_fp8(z)                        # h8 feeds the next layer's matmul_fp8
    ...
    dz, dz8 = sigmoid_bwd_fp8(z8, g)               # g: bf16
    dw = weight_grad_fp8(x8, dz)
    dx = matmul_fp8(dz8, w8, trans_b=True)

The formats, roundings and refusals are those of include/cleave_hip.h.  Everything runs on
the library's stream.
"""
from __future__ import annotations

from dataclasses import dataclass

from ._lib import call

import cleave_amd as ca

BLOCK = 128  # columns that share a scale
_SCALE_ROWS = 16


def _up(v: int, q: int) -> int:
    return (v + q - 1) // q * q


@dataclass
class Fp8Tensor:
    """A matrix in 8 bits: its codes [rows x pitch] and scales [pitch / 128 x rows up to 16].
    block_rows is the number of rows that share each scale, 1 or 128."""

    codes: "ca.Tensor"
    scales: "ca.Tensor"
    shape: tuple
    block_rows: int = 1

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes

    @property
    def args(self) -> tuple:
        """The operand as the ABI takes it."""
        return self.codes.ptr, self.codes.size, self.scales.ptr, self.scales.size


_NONE = (None, 0, None, 0)


def _matrix(t, what: str) -> tuple:
    if len(t.shape) != 2:
        raise ValueError(f"{what}: a matrix is required, got shape {tuple(t.shape)}")
    return t.shape


def _wide(dtype: str, what: str) -> str:
    if dtype not in ("f32", "bf16"):
        raise TypeError(f"{what}: expected f32 or bf16, got {dtype}")
    return dtype


def _held(t, what: str) -> "Fp8Tensor":
    if not isinstance(t, Fp8Tensor):
        raise TypeError(f"{what}: expected an Fp8Tensor, got {type(t).__name__}")
    return t


def _room(out, shape, block_rows: int, what: str) -> "Fp8Tensor":
    """out, if it can hold the result, or a new Fp8Tensor.  What out is labelled as stays until it holds that."""
    if out is None:
        return empty_fp8(shape, block_rows)
    if tuple(_held(out, what).shape) != tuple(shape):
        raise ValueError(f"{what}: out holds {tuple(out.shape)}, the result is {tuple(shape)}")
    return out


def _filled(t: "Fp8Tensor | None", block_rows: int = 1) -> "Fp8Tensor | None":
    """t, now that the library has written it with that many rows to a scale."""
    if t is not None:
        t.block_rows = block_rows
    return t


def empty_fp8(shape, block_rows: int = 1) -> Fp8Tensor:
    """Room for a matrix of that shape."""
    rows, cols = (int(d) for d in shape)
    if rows < 0 or cols < 0 or block_rows not in (1, BLOCK):
        raise ValueError(f"empty_fp8: shape {tuple(shape)}, block_rows {block_rows} (1 or {BLOCK})")
    nb = _up(cols, BLOCK) // BLOCK
    return Fp8Tensor(ca.empty((rows, nb * BLOCK), "u8"), ca.empty((nb, _up(rows, _SCALE_ROWS)), "u8"), (rows, cols),
                     block_rows)


def quantize_fp8(x, block_rows: int = 1, out: Fp8Tensor | None = None) -> Fp8Tensor:
    """x (f32 or bf16) in 8 bits: a scale for each row's 128 columns, or, with
    block_rows=128, for each 128 x 128 block (a weight)."""
    rows, cols = _matrix(x, "quantize_fp8")
    sfx = _wide(x.dtype, "quantize_fp8")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"quantize_fp8: block_rows is 1 or {BLOCK}, not {block_rows}")
    out = _room(out, (rows, cols), block_rows, "quantize_fp8")
    call(f"cleave_hip_quantize_fp8_{sfx}", x.ptr, x.size, *out.args, rows, cols, block_rows)
    return _filled(out, block_rows)


def dequantize_fp8(t: Fp8Tensor, dtype: str = "f32", out=None):
    """The values held, as an f32 or bf16 tensor."""
    rows, cols = _held(t, "dequantize_fp8").shape
    out = out if out is not None else ca.empty((rows, cols), _wide(dtype, "dequantize_fp8"))
    call(f"cleave_hip_dequantize_fp8_{_wide(out.dtype, 'dequantize_fp8')}", *t.args, out.ptr, out.size, rows, cols)
    return out


def _product_dims(shape, b: Fp8Tensor, trans_b: bool, what: str) -> tuple:
    M, K = shape
    Kb, N = (b.shape[1], b.shape[0]) if trans_b else b.shape
    if K != Kb:
        raise ValueError(f"{what}: inner dimensions differ ({K} vs {Kb})")
    if not trans_b and b.block_rows != BLOCK:
        raise ValueError(f"{what}: an operand stored K x N needs block_rows={BLOCK}: its scales may not vary along K "
                         "inside a block")
    return M, N, K


def matmul_fp8(a: Fp8Tensor, b: Fp8Tensor, trans_b: bool = False, dtype: str = "f32", out=None):
    """C = a b (b quantised with block_rows=128) or, with trans_b, a b^T, as f32 or bf16.
    bf16 results of more than 32 rows keep products to 2^-13 of the largest of 8; f32
    ones, and those of fewer rows, are f32 sums."""
    M, N, K = _product_dims(_held(a, "matmul_fp8").shape, _held(b, "matmul_fp8"), trans_b, "matmul_fp8")
    out = out if out is not None else ca.empty((M, N), _wide(dtype, "matmul_fp8"))
    call(f"cleave_hip_matmul_fp8_{_wide(out.dtype, 'matmul_fp8')}", *a.args, *b.args, out.ptr, out.size, M, N, K,
         int(trans_b))
    return out


def linear_fp8(x, w: Fp8Tensor, trans_b: bool = False, dtype: str = "f32", out=None, x8: Fp8Tensor | None = None):
    """y = Q(x) w (or Q(x) w^T), Q(x) being x quantised by rows, summed as matmul_fp8 sums;
    x8 receives Q(x), which weight_grad_fp8 reads in the backward pass."""
    M, N, K = _product_dims(_matrix(x, "linear_fp8"), _held(w, "linear_fp8"), trans_b, "linear_fp8")
    out = out if out is not None else ca.empty((M, N), _wide(dtype, "linear_fp8"))
    if x8 is not None:
        x8 = _room(x8, (M, K), 1, "linear_fp8")
    call(f"cleave_hip_linear_fp8_{_wide(x.dtype, 'linear_fp8')}_{_wide(out.dtype, 'linear_fp8')}", x.ptr, x.size,
         *w.args, out.ptr, out.size, *(x8.args if x8 is not None else _NONE), M, N, K, int(trans_b))
    _filled(x8)
    return out


def weight_grad_fp8(x8: Fp8Tensor, g, out=None):
    """dw = x^T g (f32) from the kept input x and g in bf16."""
    B, D = _held(x8, "weight_grad_fp8").shape
    rows, H = _matrix(g, "weight_grad_fp8")
    if rows != B:
        raise ValueError(f"weight_grad_fp8: {B} rows of x, {rows} of g")
    ca._need(g, "bf16", "weight_grad_fp8")
    out = out if out is not None else ca.empty((D, H))
    ca._need(out, "f32", "weight_grad_fp8")
    call("cleave_hip_weight_grad_fp8", *x8.args, g.ptr, g.size, out.ptr, out.size, B, D, H)
    return out


def _act(act: str, z, save: bool, h8: Fp8Tensor | None, z8: Fp8Tensor | None):
    what = f"{act}_fp8"
    shape = _matrix(z, what)
    sfx = _wide(z.dtype, what)
    h8 = _room(h8, shape, 1, what)
    if save or z8 is not None:
        z8 = _room(z8, shape, 1, what)
    call(f"cleave_hip_{act}_fp8_{sfx}", z.ptr, z.size, *h8.args, *(z8.args if z8 is not None else _NONE), *shape)
    return _filled(h8), _filled(z8)


def relu_fp8(z, h8: Fp8Tensor | None = None) -> Fp8Tensor:
    """relu(z) in 8 bits; its codes are the checkpoint as well (a positive h never gets the code 0)."""
    return _act("relu", z, False, h8, None)[0]


def sigmoid_fp8(z, save: bool = True, h8: Fp8Tensor | None = None, z8: Fp8Tensor | None = None):
    """(h8, z8): sigmoid(z) in 8 bits and, unless save is false, z for sigmoid_bwd_fp8."""
    return _act("sigmoid", z, save, h8, z8)


def tanh_fp8(z, save: bool = True, h8: Fp8Tensor | None = None, z8: Fp8Tensor | None = None):
    """(h8, z8): tanh(z) in 8 bits and, unless save is false, z for tanh_bwd_fp8."""
    return _act("tanh", z, save, h8, z8)


def _act_bwd(act: str, z8: Fp8Tensor, g, out, out8: Fp8Tensor | None, codes: bool):
    what = f"{act}_bwd_fp8"
    shape = _held(z8, what).shape
    if tuple(_matrix(g, what)) != tuple(shape):
        raise ValueError(f"{what}: checkpoint {tuple(shape)}, gradient {tuple(g.shape)}")
    sfx = _wide(g.dtype, what)
    out = out if out is not None else ca.empty(shape, sfx)
    ca._need(out, sfx, what)
    if codes or out8 is not None:
        out8 = _room(out8, shape, 1, what)
    call(f"cleave_hip_{act}_bwd_fp8_{sfx}", *z8.args, g.ptr, g.size, out.ptr, out.size,
         *(out8.args if out8 is not None else _NONE), *shape)
    return out, _filled(out8)


def relu_bwd_fp8(h8: Fp8Tensor, g, out=None, out8: Fp8Tensor | None = None, codes: bool = True):
    """(dz, dz8) = g where h > 0: in g's type for weight_grad_fp8, and in 8 bits for
    matmul_fp8 (unless codes is false: a first layer needs no gradient of its input).
    out may be g."""
    return _act_bwd("relu", h8, g, out, out8, codes)


def sigmoid_bwd_fp8(z8: Fp8Tensor, g, out=None, out8: Fp8Tensor | None = None, codes: bool = True):
    """(dz, dz8) = g s (1 - s), s = sigmoid(z)."""
    return _act_bwd("sigmoid", z8, g, out, out8, codes)


def tanh_bwd_fp8(z8: Fp8Tensor, g, out=None, out8: Fp8Tensor | None = None, codes: bool = True):
    """(dz, dz8) = g (1 - t^2), t = tanh(z)."""
    return _act_bwd("tanh", z8, g, out, out8, codes)

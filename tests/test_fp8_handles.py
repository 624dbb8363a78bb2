"""What a refused call leaves of the handle it was to fill: its label, which the products trust.  No GPU needed:
null pointers are refused before any device work."""
from __future__ import annotations

import pytest


def none(shape, dtype="u8"):
    import cleave_amd as ca

    return ca.Tensor(0, shape, dtype, owned=False)


def room(rows, cols, block_rows):
    import cleave_amd as ca

    up = lambda v, q: -(-v // q) * q  # noqa: E731
    return ca.Fp8Tensor(none((rows, up(cols, 128))), none((up(cols, 128) // 128, up(rows, 16))), (rows, cols), block_rows)


@pytest.mark.parametrize("held,asked", [(128, 1), (1, 128)])
def test_quantize_refused(held, asked):
    import cleave_amd as ca

    out = room(4, 256, held)
    with pytest.raises(ca.CleaveHipError, match="null"):
        ca.quantize_fp8(none((4, 256), "f32"), block_rows=asked, out=out)
    assert out.block_rows == held


def test_the_other_outputs_refused():
    import cleave_amd as ca

    x, w = none((4, 256), "bf16"), room(256, 8, 128)
    outs = [room(4, 256, 128) for _ in range(4)]
    with pytest.raises(ca.CleaveHipError, match="null"):
        ca.linear_fp8(x, w, out=none((4, 8), "f32"), x8=outs[0])
    with pytest.raises(ca.CleaveHipError, match="null"):
        ca.sigmoid_fp8(x, h8=outs[1], z8=outs[2])
    with pytest.raises(ca.CleaveHipError, match="null"):
        ca.tanh_bwd_fp8(room(4, 256, 1), x, out=none((4, 256), "bf16"), out8=outs[3])
    # a second output of the wrong shape: the first is not relabelled either
    with pytest.raises(ValueError, match="holds"):
        ca.tanh_fp8(x, h8=outs[1], z8=room(4, 255, 128))
    assert [t.block_rows for t in outs] == [128] * 4

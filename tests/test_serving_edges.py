"""Calls at the edges of the serving ops: shapes that have to be refused because a kernel would read or write past them, and operands that
are allowed but unusual. CPU backend, and marked `gpu` the kernels."""
import pytest
import torch

from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops


def test_shapes_that_do_not_fit_are_refused():
    """No shape may reach a kernel that would read or write outside a tensor: every operand is compared with the others."""
    ir = xl.Ir()
    with ir.main_graph:
        def var(shape, dt=xl.int32):
            return xl.variable(xl.LazyInit(shape, kind="zeros"), dt)

        def rules(**kw):
            shapes = dict(history=((2, 9), xl.int32), start=((2,), xl.int32), penalties=((2, 3), xl.float32), bias_tokens=((2, 4), xl.int32),
                          bias_values=((2, 4), xl.float32), allowed=((2, 2), xl.int32))
            return ops.LogitRules(*(var(*kw.get(k, s)) for k, s in shapes.items()))

        f32, bf16 = xl.float32, xl.bfloat16
        x, y = var((6, 16), f32), var((4, 16), bf16)
        assert ops.residual_rms_(x, y, var((16,), f32)).shape == (4, 16) and ops.residual_rms_(x, y) is None
        for args in ((x, var((4, 8), bf16)), (x, var((4, 24), bf16)), (x, var((7, 16), bf16)), (x, y, var((8,), f32)), (x, y, var((16,), bf16)),
                     (var((6, 16), bf16), y), (x, var((16,), bf16))):
            with pytest.raises(ValueError, match="residual stream|norm"):
                ops.residual_rms_(*args)

        plain, joint = ops.split_glu(var((3, 20), bf16), 8, 5, 7.0)
        assert plain.shape == (3, 8) and joint.shape == (3, 11)
        assert ops.split_glu(var((3, 8), bf16), 8, 5, 7.0)[1].shape == (3, 5)
        for shape, cols, lead in (((3, 21), 8, 5), ((3, 6), 8, 5), ((3, 20), -2, 5), ((3, 20), 8, -1), ((20,), 8, 5)):
            with pytest.raises(ValueError, match="gate and up"):
                ops.split_glu(var(shape, bf16), cols, lead, 7.0)

        logits, slot = var((2, 50), f32), var((2,))
        ops.shape_logits(logits, slot, slot, rules())
        for bad in (dict(bias_tokens=((1, 4), xl.int32)), dict(bias_values=((1, 4), f32)), dict(start=((1,), xl.int32)),
                    dict(allowed=((1, 2), xl.int32)), dict(penalties=((1, 3), f32)), dict(history=((3, 9), xl.int32))):
            with pytest.raises(ValueError, match="rules"):
                ops.shape_logits(logits, slot, slot, rules(**bad))
        for bad in (var((2, 50)), var((50,), f32)):
            with pytest.raises(ValueError, match="logits"):
                ops.shape_logits(bad, slot, slot, rules())
            with pytest.raises(ValueError, match="logits"):
                ops.take_shaped_(var((2,)), bad, var((4, 2)), var((1,)), slot, slot, rules())
        with pytest.raises(ValueError, match="position"):
            ops.take_shaped_(var((2,)), logits, var((4, 2)), var((2,)), slot, slot, rules())

        ops.append_tokens_(var((2, 6)), var((4,)), slot, slot, 2)
        for history, tokens in ((var((2, 6), f32), var((4,))), (var((2, 6)), var((4,), f32))):
            with pytest.raises(ValueError, match="int32"):
                ops.append_tokens_(history, tokens, slot, slot, 2)

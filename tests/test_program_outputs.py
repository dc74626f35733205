"""Outputs of captured programs: memory of their own where nothing else holds it, a copy where something does."""
import numpy as np
import pytest
import torch

from popxl_addons_b200 import xl
from popxl_addons_b200.xl import ops


def program(device, build):
    ir = xl.Ir()
    with ir.main_graph:
        v = xl.variable(np.arange(6, dtype=np.float32), xl.float32, "v")
        stream = xl.h2d_stream((6,), xl.float32, "x")
    p, outs = xl.Program(ir, "p"), []
    with p:
        for name, t in build(ops.host_load(stream), p.use(v, by_ref=True)).items():
            outs.append((name, xl.d2h_stream(t.shape, t.dtype, name)))
            ops.host_store(outs[-1][1], t)
    return xl.Session(ir, device), p, stream, dict(outs), v


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_every_kind_of_output(device):
    """A temporary, the same one twice, a view, an input, a variable, and one that is changed after it was stored."""
    def build(x, v):
        a, b = x + 1.0, x * 2.0
        out = {"fresh": a, "twice": a, "view": ops.reshape(b, (2, 3)), "input": x, "variable": v}
        return out

    session, p, stream, outs, v = program(device, build)
    for i in range(4):
        x = np.full(6, float(i), np.float32)
        got = session.run_program(p, {stream: x})
        assert np.array_equal(got[outs["fresh"]], x + 1) and np.array_equal(got[outs["twice"]], x + 1)
        assert np.array_equal(got[outs["view"]], (2 * x).reshape(2, 3)) and np.array_equal(got[outs["input"]], x)
        assert np.array_equal(got[outs["variable"]], np.arange(6))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_values_changed_after_they_were_stored(device):
    ir = xl.Ir()
    with ir.main_graph:
        v = xl.variable(np.zeros(4, np.float32), xl.float32, "v")
    p = xl.Program(ir, "p")
    with p:
        t = p.use(v, by_ref=True)
        early, late = (xl.d2h_stream((4,), xl.float32, n) for n in ("early", "late"))
        ops.host_store(early, t)
        ops.var_updates.copy_var_update_(t, t + 1.0)
        ops.host_store(late, t)
    session = xl.Session(ir, device)
    for i in range(4):
        got = session.run_program(p)
        assert (got[early] == i).all() and (got[late] == i + 1).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_called_graph_stores_what_it_returns(device):
    """The caller changes in place what the called graph stored."""
    ir = xl.Ir()
    with ir.main_graph:
        stream = xl.h2d_stream((4,), xl.float32, "x")
    p = xl.Program(ir, "p")
    with p:
        early, late = (xl.d2h_stream((4,), xl.float32, n) for n in ("early", "late"))

        def body(t):
            y = t * 2.0
            ops.host_store(early, y)
            return y

        x = ops.host_load(stream)
        y, = ops.call(ir.create_graph(body, x), x)
        ops.var_updates.accumulate_(y, x)
        ops.host_store(late, y)
    session = xl.Session(ir, device)
    for i in range(1, 5):
        got = session.run_program(p, {stream: np.full(4, float(i), np.float32)})
        assert (got[early] == 2 * i).all() and (got[late] == 3 * i).all()


@pytest.mark.gpu
def test_outputs_without_copies():
    """Copies stay as they are when the program runs again; without copies the buffers are the program's own."""
    session, p, stream, outs, _ = program("cuda", lambda x, v: {"fresh": x + 1.0})
    first = []
    for i in range(5):
        x = torch.full((6,), float(i))
        first.append(session.run_program(p, {stream: x}, fetch=False)[outs["fresh"]])
    torch.cuda.synchronize()
    assert [t.flatten()[0].item() for t in first] == [1, 2, 3, 4, 5]
    own = [session.run_program(p, {stream: torch.full((6,), float(i))}, fetch=False, copy=False)[outs["fresh"]] for i in (7, 8)]
    torch.cuda.synchronize()
    assert own[0].data_ptr() == own[1].data_ptr() and own[1].flatten()[0].item() == 9


def test_device_tensor():
    ir = xl.Ir()
    with ir.main_graph:
        v = xl.variable(np.zeros(3, np.float32), xl.float32, "v")
    session = xl.Session(ir, "cpu")
    session.device_tensor(v).copy_(torch.tensor([1.0, 2.0, 3.0]))
    assert session.get_tensor_data(v).tolist() == [1, 2, 3]
    with ir.main_graph:
        other = xl.variable(np.zeros(3, np.float32), xl.float32, "w")
    with pytest.raises(KeyError):
        session.device_tensor(other)

"""Limits of the client's token step that need no GPU: what a table may be, and what its values become."""
from types import SimpleNamespace

import pytest
import torch

ON_GPU_0 = SimpleNamespace(p=SimpleNamespace(device=0), h=None)    # a context as far as the checks of arguments look


@pytest.mark.parametrize("rows,ok", [(1 << 30, True), ((1 << 30) + 1, False), ((1 << 31) - 1, False), ((1 << 31) + 5, False)])
def test_rows_of_a_table(rows, ok):
    """The products count rows in 32 bits, rounded up to whole blocks (tensors without memory: the size alone is looked at)."""
    from fhessm import FheError
    from fhessm.client import Q4Table
    w, s = torch.empty(rows, 16, dtype=torch.uint8, device="meta"), torch.empty(rows, 1, dtype=torch.float16, device="meta")
    if ok:
        assert Q4Table(w, s, cols=32, group=32).rows == rows
    else:
        with pytest.raises(FheError, match="rows at most"):
            Q4Table(w, s, cols=32, group=32)


def test_gradients_are_refused():
    """An operand, an output or a setting that requires a gradient: refused before anything else is looked at, served where
    gradients are off (then these host tensors are refused for what they are)."""
    from fhessm import FheError, client
    w = torch.zeros(4, 32, dtype=torch.uint8)
    table = client.Q4Table(w, torch.ones(4, 2), cols=64, group=32)
    learnt = client.Q4Table(w, torch.ones(4, 2, requires_grad=True), cols=64, group=32)
    x, u, ids = torch.ones(2, 64), torch.zeros(2), torch.zeros(2, dtype=torch.int64)
    f = lambda *shape: torch.ones(*shape, requires_grad=True)
    for call in [lambda: client.q4_matvec(ON_GPU_0, f(2, 64), table), lambda: client.q4_matvec(ON_GPU_0, x, learnt),
                 lambda: client.q4_matvec(ON_GPU_0, x, table, out=f(2, 4)), lambda: client.q4_rows(ON_GPU_0, ids, learnt),
                 lambda: client.q4_rows(ON_GPU_0, ids, table, out=f(2, 64)), lambda: client.sample(ON_GPU_0, f(2, 9), u),
                 lambda: client.sample(ON_GPU_0, torch.ones(2, 9), u, temperature=f(2)),
                 lambda: client.sample(ON_GPU_0, torch.ones(2, 9), u, top_p=f(2)),
                 lambda: client.sample(ON_GPU_0, torch.ones(2, 9), u, min_p=f(2)),
                 lambda: client.sample(ON_GPU_0, torch.ones(2, 9), f(2))]:
        with pytest.raises(FheError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(FheError, match="not on the context's GPU"):
            call()


def test_quantise_takes_a_parameter():
    """The nearest table is no differentiable function of the weights: it holds none of their graph."""
    from fhessm.client import Q4Table
    w = torch.nn.Parameter(torch.randn(3, 64))
    t = Q4Table.quantise(w, group=32)
    assert not t.scale.requires_grad and torch.equal(t.weight, Q4Table.quantise(w.detach(), group=32).weight)


@pytest.mark.parametrize("value,dtype", [(float("inf"), torch.float32), (float("nan"), torch.bfloat16), (-5e5, torch.float16)])
def test_quantise_refuses_what_no_scale_holds(value, dtype):
    """A group's scale is its largest magnitude over 7: 65,504 x 7 = 458,528 is the end of float16's."""
    from fhessm import FheError
    from fhessm.client import Q4Table
    w = torch.ones(3, 100)
    w[1, 70] = value
    with pytest.raises(FheError, match="scale"):
        Q4Table.quantise(w, group=32, scale_dtype=dtype)
    w[1, 70] = 4.5e5
    t = Q4Table.quantise(w, group=32, scale_dtype=dtype)
    assert torch.isfinite(t.dequantise()).all()


def test_a_table_of_no_rows_and_sizes_that_are_no_whole_numbers():
    import numpy as np
    from fhessm import FheError
    from fhessm.client import Q4Table
    w, s = torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 2)
    assert Q4Table(w, s, cols=np.int64(64), group=np.int32(32)).cols == 64
    for kw in (dict(cols=64.0, group=32), dict(cols=64, group=32.0), dict(cols="64", group=32), dict(cols=64, group=None)):
        with pytest.raises(FheError):
            Q4Table(w, s, **kw)
    empty = Q4Table.quantise(torch.zeros(0, 70), group=32)
    assert empty.rows == 0 and empty.dequantise().shape == (0, 70)
    for kw in (dict(group=32.0), dict(group=48), dict(group=32, scale_dtype=torch.float64), dict(group=32, scale_dtype=torch.int8)):
        with pytest.raises(FheError):
            Q4Table.quantise(torch.ones(2, 64), **kw)

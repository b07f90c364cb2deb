"""CPU checks of a set of gradients that is kept over steps: what its table says after its tensors changed. The tensors
are host memory that says it is on GPU 0; nothing is launched."""
import types

import numpy as np
import pytest
import torch

import cdclq
from cdclq import tune

CTX = types.SimpleNamespace(device=0)
CODE = {torch.float32: cdclq.DTYPE_F32, torch.float16: cdclq.DTYPE_F16, torch.bfloat16: cdclq.DTYPE_BF16}


class OnGpu(torch.Tensor):
    def get_device(self):
        return 0


def make(*shape, dtype=torch.float32):
    return torch.ones(shape, dtype=dtype).as_subclass(OnGpu)


def rows(g):
    """The table as the next call takes it."""
    assert g._addresses() == g.table.ctypes.data
    return g.table


def same(row, x, out=None):
    o = x if out is None else out
    return (row["count"], row["dtype"], row["out_dtype"]) == (x.numel(), CODE[x.dtype], CODE[o.dtype]) and \
        (x.numel() == 0 or (row["x"], row["out"]) == (x.data_ptr(), o.data_ptr()))


CHANGES = {"shorter": lambda x: x.data[:10], "empty": lambda x: x.data[:0], "longer": lambda x: x.base[:1200],
           "retyped": lambda x: x.data.view(torch.bfloat16), "reshaped": lambda x: x.data.view(20, 50),
           "moved": lambda x: x.base[7:507], "other": lambda x: make(30, dtype=torch.float16)}


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("count", [1, 3, 200])
def test_a_tensor_changed_in_place_is_read_again(change, count):
    """Sizes and types at the address that the tensor had before, too."""
    tensors = [make(1000 + i) for i in range(count)]
    x = tensors[count // 2]
    x.data = (base := make(2000))[:1000]
    x.base = base
    g = tune.Gradients(CTX, tensors)
    assert all(same(r, t) for r, t in zip(rows(g), tensors))
    x.data = CHANGES[change](x)
    assert all(same(r, t) for r, t in zip(rows(g), tensors))
    assert g.work_bytes == cdclq.lib().cdclq_grad_work_bytes(g.ptr, count, 1)


def test_resized_and_refilled_tensors():
    x = make(1000)
    g = tune.Gradients(CTX, [x])
    x.resize_(400)
    assert same(rows(g)[0], x)
    for n in (300, 20, 900, 1):  # freed first: the allocator may hand out the same place
        for _ in range(20):
            x.data = make(0)
            assert same(rows(g)[0], x)
            x.data = make(n, dtype=torch.float16 if n == 20 else torch.float32)
            assert same(rows(g)[0], x)


def test_outputs_are_looked_at_as_gradients_are():
    x, out = make(6, 50, dtype=torch.float16), make(6, 50)
    g = tune.Gradients(CTX, [x], out=[out])
    assert same(rows(g)[0], x, out)
    out.data = out.data.view(torch.float16)[:, ::2].contiguous()
    assert same(rows(g)[0], x, out)
    x.data, out.data = x.data[:3], out.data[:3]
    assert same(rows(g)[0], x, out)
    out.data = out.data[:2]
    with pytest.raises(ValueError, match="shape"):
        g._addresses()
    out.data = x.data.view(3 * 50)
    with pytest.raises(ValueError, match="shape"):
        g._addresses()


def test_transposed_in_place_is_refused():
    x = make(20, 30)
    g = tune.Gradients(CTX, [x])
    x.t_()
    with pytest.raises(ValueError, match="contiguous"):
        g._addresses()
    x.t_()
    assert same(rows(g)[0], x)
    x.data = make(40, 30)[::2]
    with pytest.raises(ValueError, match="contiguous"):
        g._addresses()


def test_types_without_kernels_are_refused_later_too():
    x = make(10)
    g = tune.Gradients(CTX, [x])
    x.data = x.data.view(torch.int32)
    with pytest.raises(TypeError, match="int32"):
        g._addresses()


def test_adapters_stay_the_first_dimension():
    x = make(4, 6, 5)
    g = tune.Gradients(CTX, [x], adapters=4)
    x.data = x.data.view(4, 30)
    assert same(rows(g)[0], x)
    x.data = x.data.view(6, 20)
    with pytest.raises(ValueError, match="adapters first"):
        g._addresses()
    x.data = x.data.view(120)[:1].view(())
    with pytest.raises(ValueError, match="adapters first"):
        g._addresses()


def test_an_unchanged_set_is_not_read_again(monkeypatch):
    """Gradients of parameters, of size 0 and 1, with strides that say nothing."""
    param = torch.nn.Parameter(torch.ones(5)).as_subclass(OnGpu)
    tensors = [make(3, 4), make(0, 7), make(1, 9)[:, :1], make(), make(4, 1).transpose(0, 1), param, make(2)[1:]]
    out = [make(*t.shape) for t in tensors]
    for g in (tune.Gradients(CTX, tensors), tune.Gradients(CTX, tensors, out=out), tune.Gradients(CTX, [])):
        before = g.table.copy()
        monkeypatch.setattr(g, "_read", lambda: pytest.fail("read again"))
        assert np.array_equal(rows(g), before)


def test_a_set_without_the_exchange_interface_is_read_in_each_call(monkeypatch):
    monkeypatch.setattr(tune, "_exchange", None)
    monkeypatch.delattr(torch.Tensor, "__dlpack_c_exchange_api__")
    x = make(1000)
    g = tune.Gradients(CTX, [x])
    x.data = x.data[:10]
    assert same(rows(g)[0], x)
    x.data = x.data.view(2, 5).t()
    with pytest.raises(ValueError, match="contiguous"):
        g._addresses()
    monkeypatch.setattr(tune, "_exchange", None)


def test_a_tensor_that_cannot_be_described_is_read_again(monkeypatch):
    x = make(1000)
    g = tune.Gradients(CTX, [x])
    monkeypatch.setattr(g, "holds", lambda *_: (_ for _ in ()).throw(BufferError("no")))
    x.data = x.data[:10]
    assert same(rows(g)[0], x)


VIEWS = {"alone": lambda: [torch.ones(5), torch.ones(7)], "split": lambda: list(torch.ones(12).split([5, 7])),
         "of views": lambda: [x.view(-1, 1) for x in torch.ones(3, 12)[1:].flatten().split(12)],
         "chunks": lambda: list(torch.ones(4, 6).chunk(2)), "unbound": lambda: list(torch.ones(4, 6).unbind()),
         "detached": lambda: [torch.ones(9).detach()[2:], torch.ones(3).data],
         "unsafe": lambda: list(torch.ones(12).unsafe_split(4)), "parameters": lambda: [torch.nn.Parameter(torch.ones(4))],
         "moved": lambda: [moved(x) for x in torch.ones(12).split(6)]}


def moved(x):
    x.data = torch.zeros(3)
    return x


@pytest.mark.parametrize("kind", VIEWS)
def test_every_written_tensors_counter_is_among_the_sets(kind):
    """Tensors of buckets have one counter together."""
    tensors = VIEWS[kind]()
    for out in (None, [torch.ones_like(x) for x in tensors]):
        written = tensors if out is None else out
        g = object.__new__(tune.Gradients)
        with pytest.raises(ValueError, match="is on cpu"):  # host memory; what it writes is known by then
            g.__init__(CTX, tensors, out=out)
        for _ in range(4):
            before = [x._version for x in written]
            g._changed()
            assert all(x._version > b for x, b in zip(written, before))


def test_a_sets_own_count_is_what_a_call_takes(monkeypatch):
    """Lists that are changed after the set was made are not the set's."""
    tensors = [make(5), make(6)]
    g = tune.Gradients(CTX, tensors)
    tensors.append(make(7))
    g.tensors.append(make(8))
    monkeypatch.setattr(tune, "_empty", lambda *_, **__: None)
    assert tune._grad_call(g)[2] == len(g.table) == 2
    g.tensors[0].data = make(3)
    assert same(rows(g)[0], g.tensors[0]) and tune._grad_call(g)[2] == len(g.table) == 2


@pytest.mark.parametrize("inside", [True, False])
def test_views_of_inference_mode_are_written_without_an_error(inside):
    base = torch.ones(12)
    with torch.inference_mode():
        tensors = list((torch.ones(12) if inside else base).split(4))
    g = object.__new__(tune.Gradients)
    with pytest.raises(ValueError, match="is on cpu"):
        g.__init__(CTX, tensors)
    for _ in range(3):
        g._changed()

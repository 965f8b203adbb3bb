"""Argument checks of the soft reads, without a GPU, and the 64-bit definitions that the GPU tests compare with."""
import ctypes
import math
import os
import subprocess

import pytest

import attention_ref as R

torch = pytest.importorskip("torch")


def attend_args(fm, **over):
    a = fm.abi.AttendArgs()
    v = dict(q=64, k=64, v=64, out=64, status=64, n=10, batch=2, queries=3, heads=4, kv_heads=2, d=64, storage=2, scale=0.125)
    v.update(over)
    for name, x in v.items():
        setattr(a, name, x)
    for name in ("q_stride", "k_stride", "v_stride"):
        for i, s in enumerate((4096, 256, 64)):
            getattr(a, name)[i] = s
    return a


def test_struct_layouts(fm, tmp_path):
    # size and every field's offset as the C compiler sees them
    names = {"B200FAttendArgs": fm.abi.AttendArgs, "B200FAttendBackwardArgs": fm.abi.AttendBackwardArgs,
             "B200FAttentionMassArgs": fm.abi.AttentionMassArgs, "B200FEvictArgs": fm.abi.EvictArgs}
    lines = []
    for c, py in names.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % c)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (c, f[0]) for f in py._fields_]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "b200_flat.h"\nint main(void) {\n%s\nreturn 0;\n}\n' % "\n".join(lines))
    exe = tmp_path / "sizes"
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for py in names.values():
        want.append(ctypes.sizeof(py))
        want += [getattr(py, f[0]).offset for f in py._fields_]
    assert got == want


BAD = [dict(d=4), dict(d=60), dict(d=136), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(heads=258), dict(storage=0), dict(storage=7),
       dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(batch=-1), dict(queries=-1), dict(n=-1),
       dict(shared_n=-1)]


@pytest.mark.parametrize("over", BAD, ids=str)
def test_bad_sizes(fm, over):
    L = fm.lib()
    a = attend_args(fm, **over)
    assert L.b200f_attend_scratch_bytes(ctypes.byref(a)) == 0
    assert L.b200f_attend(ctypes.byref(a)) == fm.abi.ERR_BAD_ARG


@pytest.mark.parametrize("over", [dict(q=None), dict(q=72), dict(k=None), dict(v=40), dict(out=None), dict(status=None), dict(shared_n=5)],
                         ids=str)
def test_bad_pointers(fm, over):
    L = fm.lib()
    a = attend_args(fm, **over)
    assert L.b200f_attend_scratch_bytes(ctypes.byref(a)) > 0
    a.scratch, a.scratch_bytes = 4096, 1 << 40
    assert L.b200f_attend(ctypes.byref(a)) == fm.abi.ERR_BAD_ARG


def test_bad_strides(fm):
    L = fm.lib()
    for name in ("q_stride", "k_stride", "v_stride"):
        for i, s in ((0, -8), (1, 100), (2, 4), (1, 0), (0, 1 << 40)):
            a = attend_args(fm, scratch=4096, scratch_bytes=1 << 40)
            getattr(a, name)[i] = s
            assert L.b200f_attend(ctypes.byref(a)) == fm.abi.ERR_BAD_ARG, (name, i, s)


def test_too_large(fm):
    L = fm.lib()
    for over in (dict(n=2 ** 31 - 1), dict(batch=2 ** 20, queries=2 ** 20), dict(queries=2 ** 40), dict(shared_n=2 ** 31 - 1)):
        a = attend_args(fm, **over)
        assert L.b200f_attend(ctypes.byref(a)) == fm.abi.ERR_UNSUPPORTED


def test_null_and_nothing(fm):
    L = fm.lib()
    assert L.b200f_attend(None) == L.b200f_attend_backward(None) == L.b200f_attention_mass(None) == L.b200f_evict(None) == 1
    a = attend_args(fm, batch=0, q=None, k=None, v=None, out=None, status=None)
    assert L.b200f_attend(ctypes.byref(a)) == 0
    e = fm.abi.EvictArgs()
    for over in (dict(keep=0), dict(recent=5, keep=4), dict(recent=-1), dict(d=12), dict(kv_heads=0), dict(storage=0), dict(n=-1)):
        for name, x in dict(keep=4, recent=0, d=16, kv_heads=1, storage=1, n=8, batch=1).items():
            setattr(e, name, x)
        for name, x in over.items():
            setattr(e, name, x)
        assert L.b200f_evict(ctypes.byref(e)) == 1


def test_scratch_is_asked_for(fm):
    L = fm.lib()
    b = fm.abi.AttendBackwardArgs()
    for name, x in dict(grad_out=64, q=64, k=64, v=64, out=64, lse=64, grad_q=64, grad_k=64, grad_v=64, status=64, n=10, batch=2,
                        queries=3, heads=4, kv_heads=2, d=64, storage=2, scale=0.125).items():
        setattr(b, name, x)
    for name in ("grad_out_stride", "q_stride", "k_stride", "v_stride"):
        for i, s in enumerate((4096, 256, 64)):
            getattr(b, name)[i] = s
    need = L.b200f_attend_backward_scratch_bytes(ctypes.byref(b))
    assert need > 0
    b.scratch, b.scratch_bytes = 4096, need - 1
    assert L.b200f_attend_backward(ctypes.byref(b)) == fm.abi.ERR_SCRATCH


def test_python_refuses_what_is_not_on_a_gpu(fm):
    x = torch.zeros(1, 1, 1, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        fm.attend(x, x, x)
    with pytest.raises(TypeError):
        fm.attend_shared([1], x[0], x[0], x, x)
    with pytest.raises(ValueError):
        fm.evict(x, x, torch.zeros(1, 1, 1), None, 1)


def test_definitions_against_autograd():
    g = torch.Generator().manual_seed(0)
    q, k, v, grad = (torch.randn(2, n, h, 16, generator=g, dtype=torch.float64) for n, h in ((5, 4), (9, 2), (9, 2), (5, 4)))
    n = torch.tensor([9, 4])
    for x in (q, k, v):
        x.requires_grad_()
    out, lse, _ = R.attend(q, k, v, n)
    out.backward(grad)
    got, _ = R.backward(grad, q.detach(), k.detach(), v.detach(), n)
    for x, y in zip((q, k, v), got):
        assert torch.allclose(x.grad, y, atol=1e-12)
    # weights of a query sum to one over the keys
    m = R.mass(q.detach(), k.detach(), lse.detach(), n)
    assert torch.allclose(m.sum(-1), torch.full((2, 2), 10.0, dtype=torch.float64))


def test_scale_that_overflows_in_base_2(fm):
    L = fm.lib()
    a = attend_args(fm, scale=2.5e38)
    assert L.b200f_attend_scratch_bytes(ctypes.byref(a)) == 0
    assert L.b200f_attend(ctypes.byref(a)) == fm.abi.ERR_BAD_ARG


def test_gradient_of_neither_queries_nor_keys(fm):
    b = fm.abi.AttendBackwardArgs()
    for name, x in dict(status=64, batch=2, heads=4, kv_heads=2, d=64, storage=2, scale=0.125, scratch=4096, scratch_bytes=1 << 20).items():
        setattr(b, name, x)
    assert fm.lib().b200f_attend_backward(ctypes.byref(b)) == 0


def test_index_reads_belong_to_the_index_device(fm, monkeypatch):
    # current device 0, index on device 1: the call goes on under the index's device, before it looks at captures, streams and events
    from importlib import import_module
    A = import_module(fm.__name__ + ".attention")
    where = [0]

    class device:
        def __init__(self, i):
            self.i = i

        def __enter__(self):
            self.old, where[0] = where[0], self.i

        def __exit__(self, *_):
            where[0] = self.old

    class event:
        def record(self):
            seen.append(("event", where[0]))

    seen = []
    plan = type("plan", (), dict(index=1, proto=bytes(fm.abi.AttendArgs()), out=staticmethod(lambda: x), lse=None, what="attend"))
    x = torch.zeros(2, 64, dtype=torch.float16)
    index = type("index", (), dict(ntotal=2, d=64, storage=1, metric_type=0, _reads={}, device_rows=lambda self: 64,
                                   resources=type("r", (), dict(device=1))))()

    class plans(dict):
        def get(self, key):
            return plan

    monkeypatch.setattr(A, "_plans", plans())
    monkeypatch.setattr(A, "_run", lambda *_: seen.append(("run", where[0])))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: where[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "Event", event)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: seen.append(("capture", where[0])))
    A.attend_index(index, x, x, None, False)
    assert seen == [("capture", 1), ("run", 1), ("event", 1)]

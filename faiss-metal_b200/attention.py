"""Soft reads of stored rows (the ``b200f_attend*`` / ``b200f_attention_mass`` / ``b200f_evict`` entry points).

``B200IndexFlat.search`` reads a store the hard way: inner products with all rows, then the k largest.  A model that
attends to stored states reads them the soft way, with a softmax in the place of the selection:

``attend``           queries of a batch to keys of another length, each sequence its own
``attend_backward``  its gradient
``attend_shared``    one or a few new queries a sequence, to rows that all sequences share and to rows of their own
``attention_mass``   the weight every row received, added up
``evict``            the rows of largest weight and the most recent move to a smaller cache

All tensors are torch CUDA tensors of one device, queries, keys and values float16 or bfloat16 in the layout [batch,
rows, heads, width]; any strides whose last is 1 and whose others are multiples of 8 (0 repeats a sequence or a head).
The work is queued on torch's current stream of that device; nothing waits for it.  A device-side error (a bounded wait that ran
out) is raised by the next call after it happened, or by ``check_attention_status()``.

The functions do not record gradients: inputs that require them are refused unless gradients are off
(``torch.no_grad()``); ``attend_backward`` is the gradient.  Forward-mode tangents and tensors inside a transform of
``torch.func`` (``vmap``, ``grad``, ``jvp``) are refused.
"""
from __future__ import annotations

import ctypes
import math
from types import SimpleNamespace

from . import abi

_STORAGE = {"float16": abi.STORAGE_F16, "bfloat16": abi.STORAGE_BF16}
MAX_WIDTH = 128
MAX_GROUP = 128
MAX_SCALE = 2e38


def check_attention_status(synchronize: bool = True) -> None:
    """Raises B200Error if a device-side check of an earlier call of this module failed.  synchronize: waits for
    torch's current stream first."""
    if synchronize:
        import torch
        torch.cuda.current_stream().synchronize()
    p = _status()
    bits = p[0]
    if bits:
        p[0] = 0
        code = abi.ERR_DEVICE_WAIT if bits & 1 else abi.ERR_DEVICE_CHECK
        raise abi.B200Error(code, "an earlier attention call: " + abi.status_string(code))


_status_word = None


def _status():
    global _status_word
    if _status_word is None:
        p = abi.lib().b200f_attention_status()
        if not p:
            raise abi.B200Error(abi.ERR_NO_DEVICE, abi.status_string(abi.ERR_NO_DEVICE))
        _status_word = ctypes.cast(p, ctypes.POINTER(ctypes.c_int32))
    return _status_word


class _Check:
    """Checks one call's operands: everything about them but their addresses."""

    def __init__(self, what: str, first):
        import torch
        self.torch = torch
        self.what = what
        if not first.is_cuda:
            raise ValueError("%s: expected CUDA tensors" % what)
        self.device = first.device
        self.dtype = first.dtype
        name = str(first.dtype).replace("torch.", "")
        if name not in _STORAGE:
            raise ValueError("%s: expected float16 or bfloat16, got %s" % (what, name))
        self.storage = _STORAGE[name]

    def tensor(self, x, name: str, dims: int, dtype=None):
        if x.device != self.device:
            raise ValueError("%s: %s: on %s, expected %s" % (self.what, name, x.device, self.device))
        if x.dtype != (dtype or self.dtype):
            raise ValueError("%s: %s: expected dtype %s, got %s" % (self.what, name, dtype or self.dtype, x.dtype))
        if x.dim() != dims:
            raise ValueError("%s: %s: expected %d dimensions, got %d" % (self.what, name, dims, x.dim()))

    def shape(self, x, name: str, shape):
        if tuple(x.shape) != tuple(shape):
            raise ValueError("%s: %s: expected shape %s, got %s" % (self.what, name, tuple(shape), tuple(x.shape)))

    def rows(self, x, name: str, dims: int = 4):
        """A 16-bit operand; returns its strides but the last."""
        self.tensor(x, name, dims)
        if x.numel() and x.shape[-1] > 1 and x.stride(-1) != 1:
            raise ValueError("%s: %s: the last dimension must be dense" % (self.what, name))
        out = []
        for i in range(dims - 1):
            s = x.stride(i) if x.shape[i] > 1 else 0
            if x.numel() and (s % 8 or (s == 0 and x.shape[i] > 1 and i == max(dims - 3, 0))):
                raise ValueError("%s: %s: stride %d of dimension %d is no positive multiple of 8" % (self.what, name, s, i))
            out.append(s)
        return out

    def dense(self, x, name: str, shape, dtype):
        self.tensor(x, name, len(shape), dtype)
        self.shape(x, name, shape)
        if not x.is_contiguous():
            raise ValueError("%s: %s: must be contiguous" % (self.what, name))

    def lengths(self, x, batch: int, name: str = "key_lengths"):
        if x is not None:
            self.dense(x, name, (batch,), self.torch.int32)

    def heads(self, h: int, hk: int, d: int):
        if hk < 1 or h < 1 or h % hk or h // hk > MAX_GROUP:
            raise ValueError("%s: %d heads do not divide into groups of %d key heads (at most %d heads a group)"
                             % (self.what, h, hk, MAX_GROUP))
        if d < 8 or d > MAX_WIDTH or d % 8:
            raise ValueError("%s: width %d is no multiple of 8 up to %d" % (self.what, d, MAX_WIDTH))

    def distinct_heads(self, x, name: str, hk: int):
        if x.numel() and x.shape[2] > hk and x.stride(2) == 0:
            raise ValueError("%s: %s: query heads of one key head must not repeat" % (self.what, name))

    def scale(self, scale, d: int) -> float:
        s = 1.0 / math.sqrt(d) if scale is None else scale
        if not (0.0 < s <= MAX_SCALE):
            raise ValueError("%s: scale must be positive and at most %g" % (self.what, MAX_SCALE))
        return s

    def plan(self, args, fn: str, with_scratch: bool = True):
        """What calls of these shapes share: the argument block without addresses, the scratch they need."""
        lib = abi.lib()
        scratch = 0
        if with_scratch:
            args.status = ctypes.addressof(_status().contents)
            with self.torch.cuda.device(self.device):
                scratch = getattr(lib, fn + "_scratch_bytes")(ctypes.byref(args))
                if scratch == 0:   # sizes that the library refuses: it says which way
                    abi.check_op(getattr(lib, fn)(ctypes.byref(args)), self.what)
        return SimpleNamespace(what=self.what, proto=bytes(args), fn=getattr(lib, fn), device=self.device, dtype=self.dtype,
                               index=self.device.index, scratch=scratch)


# Plans by operator, shapes, strides, types and options; never by address.  A server meets few of them; one that meets
# many starts over.
_plans: dict = {}
_MAX_PLANS = 4096


def _keep(key, plan):
    if len(_plans) >= _MAX_PLANS:
        _plans.clear()
    _plans[key] = plan
    return plan


def _number(x):
    """An option as a plain number, as it is now: it goes into a plan's key."""
    return None if x is None else float(x)


def _look(what: str, *tensors):
    """The part of a plan's key that comes from tensors (None: not given)."""
    import torch
    forward_ad = torch.autograd.forward_ad
    grad = torch.is_grad_enabled()
    if torch._C._functorch.peek_interpreter_stack() is not None and any(
            isinstance(x, torch.Tensor) and torch._C._functorch.is_functorch_wrapped_tensor(x) for x in tensors):
        raise ValueError("%s: has no form inside torch.func transforms (vmap, grad, jvp)" % what)
    dual = forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()
    key = [what]
    for x in tensors:
        if x is None:
            key.append(None)
            continue
        if not isinstance(x, torch.Tensor):
            raise TypeError("%s: expected torch tensors, got %s" % (what, type(x).__name__))
        if grad and x.requires_grad:
            raise ValueError("%s: a tensor requires a gradient, which is not recorded; use torch.no_grad() and attend_backward"
                             % what)
        if dual and forward_ad.unpack_dual(x).tangent is not None:
            raise ValueError("%s: a tensor carries a forward-mode tangent, which is not propagated" % what)
        key.append((x.dtype, x.shape, x.stride(), x.device))
    return key


def _run(plan, args, addresses: int, unused_scratch: int = 0):
    """addresses: all 16-bit operands' addresses, or-ed."""
    import torch
    if addresses & 15:
        raise ValueError("%s: operands must lie on 16-byte boundaries" % plan.what)
    if (_status_word or _status())[0]:
        check_attention_status(synchronize=False)
    if torch._C._cuda_getDevice() != plan.index:
        with torch.cuda.device(plan.index):
            return _run(plan, args, 0, unused_scratch)
    args.stream = torch._C._cuda_getCurrentRawStream(plan.index)
    if plan.scratch > unused_scratch:
        keep = torch.empty(plan.scratch, dtype=torch.uint8, device=plan.device)
        args.scratch, args.scratch_bytes = keep.data_ptr(), plan.scratch
    status = plan.fn(ctypes.byref(args))
    if status:
        abi.check_op(status, plan.what)


def _dense_strides(shape):
    out, n = [], 1
    for s in reversed(shape):
        out.append(n)
        n *= max(int(s), 1)
    return tuple(reversed(out))


class _Output:
    """A dense output of a plan, allocated with as little work as torch asks for."""

    def __init__(self, shape, dtype, device):
        self.shape, self.strides, self.dtype, self.device = tuple(shape), _dense_strides(shape), dtype, device

    def __call__(self):
        import torch
        return torch.empty_strided(self.shape, self.strides, dtype=self.dtype, device=self.device)


_NO_SCRATCH = 256   # scratch sizes up to this are not used by attend and attention_mass


def _set(args, name, strides):
    for i, s in enumerate(strides):
        getattr(args, name)[i] = s


def _sizes(a, b, t, n, h, hk, d, storage, scale):
    a.batch, a.queries, a.n, a.heads, a.kv_heads, a.d, a.storage, a.scale = b, t, n, h, hk, d, storage, scale


def attend(q, k, v, *, key_lengths=None, scale=None, return_lse=False):
    """Cross attention: softmax(scale * q k^T) v.

    q [batch, queries, heads, width]; k, v [batch, keys, key heads, width]; query head h reads key head
    h // (heads // key heads).  key_lengths (int32 [batch], on the device): sequence b sees its first key_lengths[b]
    keys; what lies behind them has no influence.  scale: 1 / sqrt(width) by default.  Returns the output, like q, and with
    return_lse also the log of each row's sum of exponentials, float32 [batch, queries, heads].  A sequence that sees no
    key has output 0 and log-sum -inf."""
    import torch
    scale = _number(scale)
    key = tuple(_look("attend", q, k, v, key_lengths) + [scale])
    plan = _plans.get(key)
    if plan is None:
        c = _Check("attend", q)
        a = abi.AttendArgs()
        _set(a, "q_stride", c.rows(q, "q"))
        _set(a, "k_stride", c.rows(k, "k"))
        _set(a, "v_stride", c.rows(v, "v"))
        b, t, h, d = q.shape
        n, hk = k.shape[1], k.shape[2]
        c.heads(h, hk, d)
        c.shape(k, "k", (b, n, hk, d))
        c.shape(v, "v", (b, n, hk, d))
        c.lengths(key_lengths, b)
        _sizes(a, b, t, n, h, hk, d, c.storage, c.scale(scale, d))
        plan = _keep(key, c.plan(a, "b200f_attend"))
        plan.out, plan.lse = _Output(q.shape, c.dtype, c.device), _Output((b, t, h), torch.float32, c.device)
    a = abi.AttendArgs.from_buffer_copy(plan.proto)
    out = plan.out()
    lse = plan.lse() if return_lse else None
    a.q, a.k, a.v, a.out = pq, pk, pv, _ = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.key_lengths = key_lengths.data_ptr() if key_lengths is not None else None
    a.lse = lse.data_ptr() if return_lse else None
    _run(plan, a, pq | pk | pv, _NO_SCRATCH)
    return (out, lse) if return_lse else out


def attend_backward(grad_out, q, k, v, out, lse, *, key_lengths=None, scale=None):
    """Gradient of attend(): (grad_q, grad_k, grad_v), dense, of the shapes of q, k and v.

    out and lse are what attend() returned for the same q, k, v, key_lengths and scale; grad_out has the shape of out.
    Keys that no query sees get 0.  Where k or v repeat sequences or heads (stride 0), their gradients come
    for every repetition; add them up."""
    import torch
    scale = _number(scale)
    key = tuple(_look("attend_backward", grad_out, q, k, v, out, lse, key_lengths) + [scale])
    plan = _plans.get(key)
    if plan is None:
        c = _Check("attend_backward", q)
        a = abi.AttendBackwardArgs()
        _set(a, "grad_out_stride", c.rows(grad_out, "grad_out"))
        _set(a, "q_stride", c.rows(q, "q"))
        _set(a, "k_stride", c.rows(k, "k"))
        _set(a, "v_stride", c.rows(v, "v"))
        b, t, h, d = q.shape
        n, hk = k.shape[1], k.shape[2]
        c.heads(h, hk, d)
        c.shape(k, "k", (b, n, hk, d))
        c.shape(v, "v", (b, n, hk, d))
        c.shape(grad_out, "grad_out", (b, t, h, d))
        c.distinct_heads(q, "q", hk)
        c.distinct_heads(grad_out, "grad_out", hk)
        c.dense(out, "out", (b, t, h, d), c.dtype)
        c.dense(lse, "lse", (b, t, h), torch.float32)
        c.lengths(key_lengths, b)
        _sizes(a, b, t, n, h, hk, d, c.storage, c.scale(scale, d))
        plan = _keep(key, c.plan(a, "b200f_attend_backward"))
        plan.grads = [_Output(x.shape, c.dtype, c.device) for x in (q, k, v)]
    a = abi.AttendBackwardArgs.from_buffer_copy(plan.proto)
    gq, gk, gv = [make() for make in plan.grads]
    a.grad_out, a.q, a.k, a.v, a.out = pg, pq, pk, pv, po = (
        grad_out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr())
    a.lse, a.grad_q, a.grad_k, a.grad_v = lse.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr()
    a.key_lengths = key_lengths.data_ptr() if key_lengths is not None else None
    _run(plan, a, pg | pq | pk | pv | po)
    return gq, gk, gv


def attend_shared(q, shared_k, shared_v, own_k, own_v, own_lengths=None, *, scale=None, return_lse=False):
    """Attention of a batch whose sequences share a long prefix, which is read once for all of them.

    q [batch, new, heads, width]: the last `new` tokens of every sequence, one when decoding; shared_k, shared_v [prefix,
    key heads, width]; own_k, own_v [batch, rows, key heads, width], with the new tokens' rows already in them;
    own_lengths (int32 [batch], on the device): rows of each sequence, the new ones included (default: all).  Query t sees
    the whole prefix and the own rows j < own_lengths[b] - new + 1 + t (a value that is infinite or NaN in a row that only later queries see may
    reach it all the same).  Returns the output, like q, and with return_lse the log-sums
    over both parts, float32 [batch, new, heads]."""
    import torch
    scale = _number(scale)
    key = tuple(_look("attend_shared", q, shared_k, shared_v, own_k, own_v, own_lengths) + [scale])
    plan = _plans.get(key)
    if plan is None:
        c = _Check("attend_shared", q)
        a = abi.AttendArgs()
        _set(a, "q_stride", c.rows(q, "q"))
        _set(a, "shared_k_stride", c.rows(shared_k, "shared_k", 3))
        _set(a, "shared_v_stride", c.rows(shared_v, "shared_v", 3))
        _set(a, "k_stride", c.rows(own_k, "own_k"))
        _set(a, "v_stride", c.rows(own_v, "own_v"))
        b, t, h, d = q.shape
        p, hk = shared_k.shape[0], shared_k.shape[1]
        n = own_k.shape[1]
        c.heads(h, hk, d)
        c.shape(shared_k, "shared_k", (p, hk, d))
        c.shape(shared_v, "shared_v", (p, hk, d))
        c.shape(own_k, "own_k", (b, n, hk, d))
        c.shape(own_v, "own_v", (b, n, hk, d))
        c.lengths(own_lengths, b, "own_lengths")
        _sizes(a, b, t, n, h, hk, d, c.storage, c.scale(scale, d))
        a.shared_n, a.causal = p, 1
        plan = _keep(key, c.plan(a, "b200f_attend"))
        plan.out, plan.lse = _Output(q.shape, c.dtype, c.device), _Output((b, t, h), torch.float32, c.device)
    a = abi.AttendArgs.from_buffer_copy(plan.proto)
    out = plan.out()
    lse = plan.lse() if return_lse else None
    a.q, a.shared_k, a.shared_v, a.k, a.v = pq, psk, psv, pk, pv = (
        q.data_ptr(), shared_k.data_ptr(), shared_v.data_ptr(), own_k.data_ptr(), own_v.data_ptr())
    a.out = out.data_ptr()
    a.key_lengths = own_lengths.data_ptr() if own_lengths is not None else None
    a.lse = lse.data_ptr() if return_lse else None
    _run(plan, a, pq | psk | psv | pk | pv, _NO_SCRATCH)
    return (out, lse) if return_lse else out


def attention_mass(q, k, lse, *, key_lengths=None, scale=None, causal=False, mass=None):
    """Accumulated attention weight: float32 [batch, key heads, keys], `mass` (zeros by default) plus what every key got from
    the queries of its group, sum of exp(scale * q.k - lse).

    q, k, key_lengths and scale as for attend(); lse float32 [batch, queries, heads] from attend(), or from attend_shared(), for which
    k are the own rows and causal is True (query t sees j < key_lengths[b] - queries + 1 + t), or the prefix, as one
    sequence."""
    import torch
    scale = _number(scale)
    key = tuple(_look("attention_mass", q, k, lse, key_lengths, mass) + [scale, bool(causal)])
    plan = _plans.get(key)
    if plan is None:
        c = _Check("attention_mass", q)
        a = abi.AttentionMassArgs()
        _set(a, "q_stride", c.rows(q, "q"))
        _set(a, "k_stride", c.rows(k, "k"))
        b, t, h, d = q.shape
        n, hk = k.shape[1], k.shape[2]
        c.heads(h, hk, d)
        c.shape(k, "k", (b, n, hk, d))
        c.distinct_heads(q, "q", hk)
        c.dense(lse, "lse", (b, t, h), torch.float32)
        c.lengths(key_lengths, b)
        if mass is not None:
            c.dense(mass, "mass", (b, hk, n), torch.float32)
        _sizes(a, b, t, n, h, hk, d, c.storage, c.scale(scale, d))
        a.causal = 1 if causal else 0
        plan = _keep(key, c.plan(a, "b200f_attention_mass"))
        plan.out = _Output((b, hk, n), torch.float32, c.device)
    a = abi.AttentionMassArgs.from_buffer_copy(plan.proto)
    out = plan.out()
    a.q, a.k, a.lse, a.mass_out = pq, pk, _, _ = q.data_ptr(), k.data_ptr(), lse.data_ptr(), out.data_ptr()
    a.key_lengths = key_lengths.data_ptr() if key_lengths is not None else None
    a.mass_in = mass.data_ptr() if mass is not None else None
    _run(plan, a, pq | pk, _NO_SCRATCH)
    return out


def evict(k, v, mass, key_lengths=None, keep=1, *, recent=0):
    """Cuts a cache down to `keep` rows a sequence and key head: the last `recent` rows and, of those before them, the ones of
    largest mass (ties to the lower row, NaN counts as largest); all rows where there are no more than `keep`.

    k, v [batch, rows, key heads, width]; mass float32 [batch, key heads, rows]; key_lengths int32 [batch] or None.  Returns
    (k, v, mass, rows, lengths): caches of `keep` rows in the old order, zero behind the last one, their mass [batch, key heads,
    keep], the row each slot was (int32, -1 behind the last one) and the new lengths (int32 [batch])."""
    import torch
    keep, recent = int(keep), int(recent)
    key = tuple(_look("evict", k, v, mass, key_lengths) + [keep, recent])
    plan = _plans.get(key)
    if plan is None:
        c = _Check("evict", k)
        a = abi.EvictArgs()
        _set(a, "k_stride", c.rows(k, "k"))
        _set(a, "v_stride", c.rows(v, "v"))
        b, n, hk, d = k.shape
        c.shape(v, "v", (b, n, hk, d))
        if hk < 1 or d < 8 or d > 1024 or d % 8:
            raise ValueError("evict: width %d of %d key heads: expected a multiple of 8 up to 1024, and a head" % (d, hk))
        if keep < 1 or recent < 0 or recent > keep:
            raise ValueError("evict: expected keep >= 1 and 0 <= recent <= keep, got %d and %d" % (keep, recent))
        c.dense(mass, "mass", (b, hk, n), torch.float32)
        c.lengths(key_lengths, b)
        a.batch, a.n, a.kv_heads, a.d, a.storage, a.keep, a.recent = b, n, hk, d, c.storage, keep, recent
        plan = _keep(key, c.plan(a, "b200f_evict", with_scratch=False))
        plan.outs = [_Output((b, a.keep, hk, d), c.dtype, c.device)] * 2 + [
            _Output((b, hk, a.keep), torch.float32, c.device), _Output((b, hk, a.keep), torch.int32, c.device),
            _Output((b,), torch.int32, c.device)]
    a = abi.EvictArgs.from_buffer_copy(plan.proto)
    out_k, out_v, out_mass, out_rows, out_lengths = [make() for make in plan.outs]
    a.k, a.v, a.mass = pk, pv, _ = k.data_ptr(), v.data_ptr(), mass.data_ptr()
    a.key_lengths = key_lengths.data_ptr() if key_lengths is not None else None
    a.out_k, a.out_v, a.out_mass, a.out_rows, a.out_lengths = (
        out_k.data_ptr(), out_v.data_ptr(), out_mass.data_ptr(), out_rows.data_ptr(), out_lengths.data_ptr())
    _run(plan, a, pk | pv)
    return out_k, out_v, out_mass, out_rows, out_lengths


def attend_index(index, x, values, scale, return_lse):
    """B200IndexFlat.attend()."""
    import torch
    scale = _number(scale)
    n, d = index.ntotal, index.d
    key = tuple(_look("attend", x, values) + [scale, n, d, index.storage, index.metric_type, index.resources.device])
    plan = _plans.get(key)
    if plan is None:
        c = _Check("attend", x)
        if index.metric_type != abi.METRIC_INNER_PRODUCT:
            raise ValueError("attend: the index must be one of inner products")
        if index.storage != c.storage:
            raise ValueError("attend: x must have the index's storage type (float16 or bfloat16), got %s" % c.dtype)
        if c.device.index != index.resources.device:
            raise ValueError("attend: x is on %s, the index on device %d" % (c.device, index.resources.device))
        a = abi.AttendArgs()
        xs, vs = c.rows(x, "x", 2), c.rows(values, "values", 2)
        c.shape(x, "x", (x.shape[0], d))
        c.shape(values, "values", (n, d))
        c.heads(1, 1, d)
        a.q_stride[1] = xs[0]
        a.k_stride[1], a.v_stride[1] = d, vs[0]   # 16-bit rows of an inner-product index lie side by side
        _sizes(a, 1, x.shape[0], n, 1, 1, d, c.storage, c.scale(scale, d))
        plan = _keep(key, c.plan(a, "b200f_attend"))
        plan.out, plan.lse = _Output(x.shape, c.dtype, c.device), _Output(x.shape[:1], torch.float32, c.device)
    if torch._C._cuda_getDevice() != plan.index:   # streams, captures and events below are those of the index's device
        with torch.cuda.device(plan.index):
            return attend_index(index, x, values, scale, return_lse)
    if torch.cuda.is_current_stream_capturing():
        raise ValueError("attend: the rows of an index may move, a graph cannot hold their address")
    a = abi.AttendArgs.from_buffer_copy(plan.proto)
    out = plan.out()
    lse = plan.lse() if return_lse else None
    a.q, a.k, a.v, a.out = px, _, pv, _ = x.data_ptr(), index.device_rows(), values.data_ptr(), out.data_ptr()
    a.lse = lse.data_ptr() if return_lse else None
    _run(plan, a, px | pv, _NO_SCRATCH)
    # adds and resets run on the index's own stream, and have completed when they return; the next one waits for this read
    event = index._reads.get(a.stream)
    if event is None:
        event = index._reads[a.stream] = torch.cuda.Event()
    event.record()
    return (out, lse) if return_lse else out

"""Operators of a state-space language-model block over packed residue rows (include/mdfri.h "Operators of a state-space language-model block"):

    causal_conv      the short causal convolution along every sequence
    selective_scan   the recurrence  H <- exp(D a) H + D x (x) b,  y = H c + d x  along every sequence
    selective_step   both for ONE token of each of many sequences, in one launch
    block_norm       the norms before and after a block with its gate, residual scale and residual

They stand beside the recurrent and convolutional sequence models of this package (mDeepFRI.predict: LSTM branch, CNN) for features of a block
    x -> pre-norm -> in-projection -> causal_conv -> selective_scan -> block_norm(gate=z, gate_first=True) -> out-projection -> block_norm(residual=...)
whose two projections are products of the caller's.  The reference has nothing of the kind; inference only: a tensor that asks for a gradient
or carries a tangent is refused.

Tensors are torch tensors on one GPU; work is enqueued on that GPU's current stream and nothing waits for it.  Rows of no sequence and
of a skipped one are left as they were in an `out` that is handed in and are zero in one that is made here.  Outputs are f32, bfloat16 or float16 like their
inputs, everything in between is f32."""
from __future__ import annotations

import ctypes
import operator
import struct
from ctypes import c_float, c_int32, c_int64, c_void_p

import numpy as np

from . import _hip
from .batch import _torch

ACTS = {"none": 0, "silu": 1, "sigmoid": 2}


class _Rows(ctypes.Structure):
    _fields_ = [("lengths", c_void_p), ("row_off", c_void_p), ("slots", c_void_p), ("positions", c_void_p), ("R", c_int64), ("B", c_int32), ("max_len", c_int32),
                ("n_slots", c_int32)]


class _Conv(ctypes.Structure):
    _fields_ = [("rows", _Rows), ("x", c_void_p), ("weight", c_void_p), ("bias", c_void_p), ("state", c_void_p), ("out", c_void_p), ("ldx", c_int64), ("ldo", c_int64),
                ("channels", c_int32), ("width", c_int32), ("dtype", c_int32), ("silu", c_int32), ("zero_skipped", c_int32)]


class _Scan(ctypes.Structure):
    _fields_ = [("rows", _Rows), ("x", c_void_p), ("b", c_void_p), ("c", c_void_p), ("dt", c_void_p), ("a", c_void_p), ("d", c_void_p), ("dt_bias", c_void_p), ("state", c_void_p),
                ("y", c_void_p), ("ldx", c_int64), ("ldb", c_int64), ("ldc", c_int64), ("lddt", c_int64), ("ldy", c_int64), ("heads", c_int32), ("groups", c_int32),
                ("head_dim", c_int32), ("state_dim", c_int32), ("dtype", c_int32), ("dt_dtype", c_int32), ("zero_skipped", c_int32)]


class _Step(ctypes.Structure):
    _fields_ = [("xbc", c_void_p), ("dt", c_void_p), ("conv_weight", c_void_p), ("conv_bias", c_void_p), ("a", c_void_p), ("d", c_void_p), ("dt_bias", c_void_p),
                ("conv_state", c_void_p), ("state", c_void_p), ("slots", c_void_p), ("positions", c_void_p), ("y", c_void_p), ("ldx", c_int64), ("lddt", c_int64), ("ldy", c_int64),
                ("B", c_int32), ("n_slots", c_int32), ("heads", c_int32), ("groups", c_int32), ("head_dim", c_int32), ("state_dim", c_int32), ("width", c_int32), ("dtype", c_int32),
                ("dt_dtype", c_int32), ("zero_skipped", c_int32)]


class _Norm(ctypes.Structure):
    _fields_ = [("s", c_void_p), ("gate", c_void_p), ("residual", c_void_p), ("post_weight", c_void_p), ("post_bias", c_void_p), ("pre_weight", c_void_p), ("pre_bias", c_void_p),
                ("scale_vec", c_void_p), ("residual_out", c_void_p), ("out", c_void_p), ("lds", c_int64), ("ldg", c_int64), ("ldr", c_int64), ("ldro", c_int64), ("ldo", c_int64),
                ("rows", c_int64), ("dim", c_int32), ("groups", c_int32), ("dtype", c_int32), ("residual_dtype", c_int32), ("gate_act", c_int32), ("gate_first", c_int32),
                ("center", c_int32), ("scale", c_float), ("eps", c_float)]


_DTYPES = None


def _dtype(t, name: str) -> int:
    global _DTYPES
    if _DTYPES is None:
        torch = _torch()
        _DTYPES = {torch.float32: _hip.DT_F32, torch.bfloat16: _hip.DT_BF16, torch.float16: _hip.DT_F16}
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name}: {t.dtype} is not float32, bfloat16 or float16")
    return code


class SequenceRows:
    """Which rows belong to which sequence: `lengths` (B) and `row_off` (B+1), int32 device tensors, row_off ascending, and the longest length.
    `dense`: the caller's word that the sequences leave out no row of the first `total` (None: of any array that they are used with), whose outputs then need no
    zeros when they are made here.  `build` makes one from host lengths, checks them and knows both.  The values in the tensors may change from call to call, max_len and
    `dense` with them (a graph that is replayed with other lengths wants dense=False); another number of sequences is another SequenceRows."""

    __slots__ = ("_lengths", "_row_off", "max_len", "dense", "total", "_count", "_form")
    lengths, row_off, count, form = (property(operator.attrgetter("_" + name)) for name in ("lengths", "row_off", "count", "form"))   # not to be set: they were checked together

    def __init__(self, lengths, row_off, max_len: int, dense: bool = False, total: int | None = None):
        torch = _torch()
        if lengths.dtype != torch.int32 or row_off.dtype != torch.int32 or lengths.dim() != 1 or row_off.dim() != 1 or not lengths.is_contiguous() or not row_off.is_contiguous():
            raise ValueError("lengths and row_off must be contiguous one-dimensional int32 tensors")
        if row_off.shape[0] != lengths.shape[0] + 1:
            raise ValueError(f"row_off has {row_off.shape[0]} entries for {lengths.shape[0]} sequences (one more is wanted)")
        if lengths.device != row_off.device or max_len < 0:
            raise ValueError("lengths and row_off lie on different devices, or max_len is negative")
        self._lengths, self._row_off, self.max_len, self.dense, self.total, self._count = lengths, row_off, int(max_len), dense, total, lengths.shape[0]
        self._form = (self._count, lengths.get_device())

    @classmethod
    def build(cls, lengths, device="cuda", align: int = 1):
        """From host lengths; `align` rounds every sequence's first row up (_hip: MDF_GROUP_ROWS = 16 gives the rows of mdf_layout_rows)."""
        torch = _torch()
        n = np.asarray(lengths, dtype=np.int64)
        if n.ndim != 1 or (n < 0).any() or align < 1:
            raise ValueError("lengths must be a list of counts, none negative")
        off = np.zeros(len(n) + 1, dtype=np.int64)
        np.cumsum(-(-n // align) * align, out=off[1:])
        if off[-1] >= 2**31:
            raise ValueError("too many rows for int32 offsets; split the batch")
        return cls(torch.from_numpy(n.astype(np.int32)).to(device), torch.from_numpy(off.astype(np.int32)).to(device), int(n.max(initial=0)), dense=bool(off[-1] == n.sum()), total=int(off[-1]))


def check_slots(slots, n_slots: int, device="cuda"):
    """Host list of state slots -> int32 device tensor; refuses one that is named twice or lies outside the pool (negative ones, which skip
    their sequence, may repeat)."""
    torch = _torch()
    s = np.asarray(slots, dtype=np.int64)
    live = s[s >= 0]
    if s.ndim != 1 or (live >= n_slots).any():
        raise ValueError(f"a slot lies outside the {n_slots} states")
    if len(np.unique(live)) != len(live):
        raise ValueError("two sequences share a state slot")
    return torch.from_numpy(s.astype(np.int32)).to(device)


def _matrix(t, name: str, device, tail: tuple, rows=None):
    """Checks a tensor of `rows` rows whose trailing dimensions are `tail`, contiguous inside a row; returns its row stride."""
    if not t.is_cuda:
        raise ValueError(f"{name} is not on a GPU")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.requires_grad and _torch().is_grad_enabled():
        raise ValueError(f"{name} asks for a gradient: the state-space operators are inference only")
    if tuple(t.shape[1:]) != tail or (rows is not None and t.shape[0] != rows):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, wanted {(rows if rows is not None else '*',) + tail}")
    want = 1
    for size, stride in zip(reversed(tail), reversed(t.stride()[1:])):
        if size != 1 and stride != want:
            raise ValueError(f"{name}: strides {t.stride()}: only the row stride is free")
        want *= size
    return t.stride(0)


def _vector(t, name: str, device, shape: tuple):
    """Checks an f32 parameter; returns its address (None: NULL)."""
    if t is None:
        return None
    if t.dtype != _torch().float32 or tuple(t.shape) != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape {shape} on {device}, not {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.requires_grad and _torch().is_grad_enabled():
        raise ValueError(f"{name} asks for a gradient: the state-space operators are inference only")
    return t.data_ptr()


def _indices(t, name: str, device, count: int):
    if t is None:
        return None
    if t.dtype != _torch().int32 or t.shape != (count,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {count} entries on {device}")
    return t.data_ptr()


def _state(t, name: str, device, dtype, tail: tuple, count: int):
    if t.dtype != dtype or tuple(t.shape[1:]) != tail or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {('*',) + tail} on {device}, not {t.dtype} {tuple(t.shape)} on {t.device}")
    if count and not t.shape[0]:                   # (its address is none: the library would take it for a call without states)
        raise ValueError(f"{name} has no slot for any of {count} sequences")
    if t.requires_grad and _torch().is_grad_enabled():
        raise ValueError(f"{name} asks for a gradient: the state-space operators are inference only")


def _check_rows(r: _Rows, rows: SequenceRows, device, total: int, slots, positions, state) -> None:
    if state is None and (slots is not None or positions is not None):
        raise ValueError("slots and positions belong to a kept state: none is given")
    if rows.lengths.device != device or rows.row_off.device != device:
        raise ValueError(f"lengths are on {rows.lengths.device}, not on {device}")
    n = rows.lengths.shape[0]
    _indices(slots, "slots", device, n), _indices(positions, "positions", device, n)
    r.R, r.B, r.n_slots = total, n, 0 if state is None else state.shape[0]


# What a call's checks find -- the strides, sizes and types of its argument structure -- hangs on the tensors' shapes, strides, types and devices alone, so it is
# kept by those: the checks of a decoding step cost more than its kernel.  Addresses are filled in at every call, in front of what is kept.
_KNOWN = ([], [], [], [])                          # per entry point: the (form, tail) of its latest kinds of calls


def _form(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device(), t.requires_grad)


def _flat(t):
    """The form of a tensor that has to be contiguous."""
    return None if t is None else (t.shape, t.is_contiguous(), t.dtype, t.get_device(), t.requires_grad)


def _known(entry: int, form, check):
    recent = _KNOWN[entry]
    for known, tail in recent:                     # compared, not hashed: unequal forms part at their first entries
        if known == form:
            return tail
    tail = check()
    recent.insert(0, (form, tail))
    del recent[16:]
    return tail


def _number(v, name: str, kind=lambda v: c_float(v).value):
    """A number of the host as it is now, in float32; one that lies on a GPU would have to be waited for."""
    if getattr(v, "is_cuda", False):
        raise ValueError(f"{name} is a tensor on {v.device}: a number on the host is wanted (nothing here waits for the GPU)")
    return kind(v)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _grad() -> bool:
    return _torch().is_grad_enabled()


def _dual_level() -> bool:
    """Whether forward-mode derivatives are being taken (a private name: without it the tensors are asked at every call)."""
    return getattr(_torch().autograd.forward_ad, "_current_level", 0) >= 0


def _refuse_tangents(**tensors) -> None:
    """Forward-mode derivatives, which requires_grad does not show.  At every call: a tangent is no part of a tensor's form."""
    for name, t in tensors.items():
        if t is not None and _torch().autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} carries a tangent: the state-space operators are inference only")


def _made(out, like, rows: SequenceRows, shape):
    """(`zero_skipped` is set for an output made here, so one whose every row is a sequence's needs no zeros)"""
    if out is not None:
        return out
    return like.new_empty(shape) if rows.dense and rows.total in (None, shape[0]) else like.new_zeros(shape)


def _check_out(out, like) -> None:
    if out is not None and out.dtype != like.dtype:
        raise ValueError(f"out is {out.dtype}, the input {like.dtype}")


def _call(fn, device, *args) -> None:
    """Runs a library entry on the device's current stream, with that device current."""
    cuda = _torch().cuda
    stream = cuda.current_stream(device).cuda_stream
    if cuda.current_device() == device.index:
        rc = fn(*args, stream)
    else:
        with cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        _hip.check(rc)


_ROWS = "4Qqiii4x"                                 # mdf_seq_rows
_CONV, _SCAN, _STEP, _NORM = (struct.Struct(f) for f in (_ROWS + "5Q", _ROWS + "9Q", "12Q", "10Q"))   # up to the last address of each structure
_SCALES = struct.Struct("2f4x")                    # mdf_block_norm_args' end: values, so packed at every call like the addresses


def causal_conv(x, weight, rows: SequenceRows, *, bias=None, silu: bool = True, state=None, slots=None, positions=None, out=None):
    """out[t, c] = act(bias[c] + sum_k weight[k, c] x[t - (width-1) + k, c]) along every sequence; inputs before a sequence's first token are 0.

    x (R, channels), any row stride; weight (width, channels) and bias (channels) f32, width 1..8; silu: the activation, or none.  state
    (n_slots, width, channels) of x's type keeps the last inputs (token t at entry t mod width) from call to call: `slots` (B) says which one
    each sequence owns (default: its own number), `positions` (B) how many tokens it had before (default 0: a new sequence)."""
    if _dual_level():
        _refuse_tangents(x=x, weight=weight, bias=bias, state=state, out=out)
    device = x.device

    def check():
        a = _Conv()
        code, channels, width = _dtype(x, "x"), x.shape[-1], weight.shape[0]
        a.ldx = _matrix(x, "x", device, (channels,))
        _vector(weight, "weight", device, (width, channels)), _vector(bias, "bias", device, (channels,))
        _check_rows(a.rows, rows, device, x.shape[0], slots, positions, state)
        if state is not None:
            _state(state, "state", device, x.dtype, (width, channels), rows.count)
        _check_out(out, x)
        a.ldo = channels if out is None else _matrix(out, "out", device, (channels,), x.shape[0])
        a.channels, a.width, a.dtype, a.silu, a.zero_skipped = channels, width, code, bool(silu), out is None
        return bytes(a)[_CONV.size:]

    tail = _known(0, (_form(x), _flat(weight), _flat(bias), rows.form, _flat(state), _flat(slots), _flat(positions), _form(out), bool(silu), _grad()), check)
    out = _made(out, x, rows, x.shape)
    _call(_hip.lib().mdf_causal_conv_dev, device,
          _CONV.pack(rows.lengths.data_ptr(), rows.row_off.data_ptr(), _ptr(slots), _ptr(positions), x.shape[0], rows.count, rows.max_len, 0 if state is None else state.shape[0],
                     x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(state), out.data_ptr()) + tail)
    return out


def selective_scan(x, dt, a, b, c, rows: SequenceRows, *, d=None, dt_bias=None, state=None, slots=None, positions=None, out=None):
    """With D = softplus(dt[t, h] + dt_bias[h]):  H <- exp(D a[h]) H + D x[t, h, :] (x) b[t, g, :],  y[t, h, :] = H c[t, g, :] + d[h] x[t, h, :].

    x and the result (R, heads, head_dim), dt (R, heads), b and c (R, groups, state_dim) -- views into one wider array are fine, only the
    row strides are free; a, d, dt_bias (heads) f32.  head_dim 1..256, state_dim 1..128, heads a multiple of groups.  state (n_slots, heads,
    head_dim, state_dim) f32 is continued where positions > 0 and left behind for the next call; slots / positions as in causal_conv.
    dt = -infinity masks a token whose x and b are finite: the state passes it unchanged (y still holds H c + d x).  Long sequences may be cut and summed
    in another order in another batch: the same to float32 rounding."""
    if _dual_level():
        _refuse_tangents(x=x, dt=dt, a=a, b=b, c=c, d=d, dt_bias=dt_bias, state=state, out=out)
    device = x.device

    def check():
        if x.dim() != 3 or b.dim() != 3 or dt.dim() != 2:
            raise ValueError(f"x, b, dt have {x.dim()}, {b.dim()}, {dt.dim()} dimensions, wanted 3, 3, 2")
        total, heads, head_dim = x.shape
        groups, state_dim = b.shape[1:]
        g = _Scan()
        g.dtype, g.dt_dtype = _dtype(x, "x"), _dtype(dt, "dt")
        if b.dtype != x.dtype or c.dtype != x.dtype:
            raise ValueError(f"x, b, c are {x.dtype}, {b.dtype}, {c.dtype}: one type is wanted")
        g.ldx, g.lddt = _matrix(x, "x", device, (heads, head_dim)), _matrix(dt, "dt", device, (heads,), total)
        g.ldb, g.ldc = _matrix(b, "b", device, (groups, state_dim), total), _matrix(c, "c", device, (groups, state_dim), total)
        for name, v in (("a", a), ("d", d), ("dt_bias", dt_bias)):
            _vector(v, name, device, (heads,))
        _check_rows(g.rows, rows, device, total, slots, positions, state)
        if state is not None:
            _state(state, "state", device, _torch().float32, (heads, head_dim, state_dim), rows.count)
        _check_out(out, x)
        g.ldy = heads * head_dim if out is None else _matrix(out, "out", device, (heads, head_dim), total)
        g.heads, g.groups, g.head_dim, g.state_dim, g.zero_skipped = heads, groups, head_dim, state_dim, out is None
        return bytes(g)[_SCAN.size:]

    tail = _known(1, (_form(x), _form(dt), _flat(a), _form(b), _form(c), rows.form, _flat(d), _flat(dt_bias), _flat(state), _flat(slots), _flat(positions), _form(out), _grad()), check)
    out = _made(out, x, rows, x.shape)
    args = _SCAN.pack(rows.lengths.data_ptr(), rows.row_off.data_ptr(), _ptr(slots), _ptr(positions), x.shape[0], rows.count, rows.max_len, 0 if state is None else state.shape[0],
                      x.data_ptr(), b.data_ptr(), c.data_ptr(), dt.data_ptr(), a.data_ptr(), _ptr(d), _ptr(dt_bias), _ptr(state), out.data_ptr()) + tail
    L = _hip.lib()
    need = L.mdf_scan_workspace_bytes(args)
    work = _torch().empty(need, dtype=_torch().uint8, device=device) if need else None
    _call(L.mdf_selective_scan_dev, device, args, _ptr(work), need)
    return out


def selective_step(xbc, dt, a, *, conv_weight, conv_state, state, positions=None, slots=None, conv_bias=None, d=None, dt_bias=None, out=None):
    """One token of each of B sequences: causal_conv (silu) of xbc = [x | b | c] (B, heads*head_dim + 2*groups*state_dim), then selective_scan,
    in one launch; conv_state (n_slots, width, channels) and state (n_slots, heads, head_dim, state_dim) are updated in place.  Returns y
    (B, heads, head_dim).  The caller adds 1 to the positions of the sequences it continues."""
    if _dual_level():
        _refuse_tangents(xbc=xbc, dt=dt, a=a, conv_weight=conv_weight, conv_state=conv_state, state=state, conv_bias=conv_bias, d=d, dt_bias=dt_bias, out=out)
    device = xbc.device

    def check():
        if state.dim() != 4 or xbc.dim() != 2:
            raise ValueError(f"state and xbc have {state.dim()}, {xbc.dim()} dimensions, wanted 4, 2")
        n, channels = xbc.shape
        heads, head_dim, state_dim = state.shape[1:]
        groups, odd = divmod(channels - heads * head_dim, 2 * state_dim) if state_dim else (0, 1)
        if odd or groups < 1:
            raise ValueError(f"xbc has {channels} channels: wanted {heads} x {head_dim} and twice a multiple of {state_dim}")
        width = conv_weight.shape[0]
        g = _Step()
        g.dtype, g.dt_dtype = _dtype(xbc, "xbc"), _dtype(dt, "dt")
        g.ldx, g.lddt = _matrix(xbc, "xbc", device, (channels,)), _matrix(dt, "dt", device, (heads,), n)
        _vector(conv_weight, "conv_weight", device, (width, channels)), _vector(conv_bias, "conv_bias", device, (channels,))
        for name, v in (("a", a), ("d", d), ("dt_bias", dt_bias)):
            _vector(v, name, device, (heads,))
        _state(conv_state, "conv_state", device, xbc.dtype, (width, channels), n)
        _state(state, "state", device, _torch().float32, (heads, head_dim, state_dim), n)
        if conv_state.shape[0] != state.shape[0]:
            raise ValueError(f"{conv_state.shape[0]} convolution states beside {state.shape[0]} scan states")
        _indices(slots, "slots", device, n), _indices(positions, "positions", device, n)
        _check_out(out, xbc)
        g.ldy = heads * head_dim if out is None else _matrix(out, "out", device, (heads, head_dim), n)
        g.B, g.n_slots, g.heads, g.groups, g.head_dim, g.state_dim, g.width, g.zero_skipped = n, state.shape[0], heads, groups, head_dim, state_dim, width, out is None
        return bytes(g)[_STEP.size:]

    tail = _known(2, (_form(xbc), _form(dt), _flat(a), _flat(conv_weight), _flat(conv_state), _flat(state), _flat(positions), _flat(slots), _flat(conv_bias), _flat(d), _flat(dt_bias),
                      _form(out), _grad()), check)
    if out is None:
        out = xbc.new_empty((xbc.shape[0],) + state.shape[1:3])
    _call(_hip.lib().mdf_selective_step_dev, device,
          _STEP.pack(xbc.data_ptr(), dt.data_ptr(), conv_weight.data_ptr(), _ptr(conv_bias), a.data_ptr(), _ptr(d), _ptr(dt_bias), conv_state.data_ptr(), state.data_ptr(), _ptr(slots),
                     _ptr(positions), out.data_ptr()) + tail)
    return out


def block_norm(s, *, residual=None, gate=None, gate_act: str = "silu", gate_first: bool = False, post_weight=None, post_bias=None, groups: int = 1, scale: float = 1.0,
               scale_vec=None, pre_weight=None, pre_bias=None, eps: float = 1e-6, center: bool = False, residual_out=None, out=None):
    """The norms before and after a block with its gate, residual scale and residual, in one pass over the rows of s (rows, dim):

        v = s [* act(gate), with gate_first];  v = post(v) where post_weight is given;  v = v * act(gate) where the gate comes last
        r = residual + scale * scale_vec * v  where a residual is given;  out = pre(r) where pre_weight is given

    Returns (r or None, out or None); without a residual out is v, or pre(v).  post / pre: x / sqrt(mean(x^2) + eps) * weight + bias, of x less its
    mean with `center`; post on each of `groups` equal parts of a row.  scale, eps and groups are numbers on the host.  s and gate share a type; the residual
    is float32 or of that type, and r has its type.  residual_out may be the residual itself, out may be s or the gate."""
    if _dual_level():
        _refuse_tangents(s=s, residual=residual, gate=gate, post_weight=post_weight, post_bias=post_bias, scale_vec=scale_vec, pre_weight=pre_weight, pre_bias=pre_bias, residual_out=residual_out, out=out)
    device = s.device
    has_out = pre_weight is not None or residual is None
    scale, eps, groups = _number(scale, "scale"), _number(eps, "eps"), _number(groups, "groups", operator.index)

    def check():
        if s.dim() != 2:
            raise ValueError(f"s has {s.dim()} dimensions, wanted 2")
        if gate_act not in ACTS:
            raise ValueError(f"gate_act {gate_act!r} is none of {sorted(ACTS)}")
        rows, dim = s.shape
        g = _Norm()
        g.dtype, g.lds = _dtype(s, "s"), _matrix(s, "s", device, (dim,))
        if gate is not None:
            if gate.dtype != s.dtype:
                raise ValueError(f"gate is {gate.dtype}, s {s.dtype}")
            g.ldg = _matrix(gate, "gate", device, (dim,), rows)
        for name, v in (("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight), ("pre_bias", pre_bias), ("scale_vec", scale_vec)):
            _vector(v, name, device, (dim,))
        if residual is not None:
            g.residual_dtype, g.ldr, g.ldro = _dtype(residual, "residual"), _matrix(residual, "residual", device, (dim,), rows), dim
            if residual_out is not None:
                if residual_out.dtype != residual.dtype:
                    raise ValueError(f"residual_out is {residual_out.dtype}, the residual {residual.dtype}")
                g.ldro = _matrix(residual_out, "residual_out", device, (dim,), rows)
        elif residual_out is not None:
            raise ValueError("residual_out without a residual")
        if out is not None and not has_out:
            raise ValueError("out without a pre-norm beside a residual: there is nothing to write there")
        _check_out(out, s)
        g.ldo = dim if out is None else _matrix(out, "out", device, (dim,), rows)
        g.rows, g.dim, g.groups, g.gate_act, g.gate_first, g.center = rows, dim, groups, ACTS[gate_act], bool(gate_first), bool(center)
        return bytes(g)[_NORM.size:_Norm.scale.offset]

    tail = _known(3, (_form(s), _form(residual), _form(gate), gate_act, bool(gate_first), _flat(post_weight), _flat(post_bias), groups, _flat(scale_vec), _flat(pre_weight),
                      _flat(pre_bias), bool(center), _form(residual_out), _form(out), _grad()), check)
    if residual_out is None and residual is not None:
        residual_out = residual.new_empty(s.shape)
    if out is None and has_out:
        out = s.new_empty(s.shape)
    _call(_hip.lib().mdf_block_norm_dev, device,
          _NORM.pack(s.data_ptr(), _ptr(gate), _ptr(residual), _ptr(post_weight), _ptr(post_bias), _ptr(pre_weight), _ptr(pre_bias), _ptr(scale_vec), _ptr(residual_out), _ptr(out)) + tail
          + _SCALES.pack(scale, eps))
    return residual_out, out

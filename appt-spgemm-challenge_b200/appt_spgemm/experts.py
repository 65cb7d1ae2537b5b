"""Routed products: a sparse matrix with top_k entries per row (the choice of top_k of a number of
experts for every token) times dense matrices, and the experts' products in 8 bits.

    ids --Route--> expert_ptr, row_pair, pair_row          the pairs sorted by expert
    x   --Dispatch / DispatchQuantize--> sorted rows       (gradient: Combine)
    rows --ScaledProduct--> rows                           each expert's own matrix
    rows --Quantize--> rows in 8 bits                      plain, or silu(gate) * up
    rows --Combine--> tokens                               (gradient: CombineGrad)

Each class builds the arguments of one library call once; ``run(stream)`` makes the call, as often
as wanted, on the buffers' present contents. Calls are asynchronous on ``stream`` (a CUDA stream
handle as an int, e.g. ``torch.cuda.current_stream().cuda_stream``; None: the device's default
stream), allocate nothing and may be captured into CUDA graphs. The C entry points
(include/appt_spgemm.h, "Routed products") define each operation and check every argument; an
``ApptError`` says what was refused.

Operands are objects with ``data_ptr()``, ``shape``, ``stride()``, ``dtype`` and ``device`` (torch
tensors; this module imports no torch) or ``Dense`` descriptions of raw device pointers. The
objects are kept alive as long as the call is. No counterpart in the reference.
"""
from __future__ import annotations

import ctypes as ct

from . import ApptError, _check, load

TYPES = {"f64": 0, "f32": 1, "f16": 2, "bf16": 3, "e4m3": 4, "i32": 5, "i64": 6}
_DTYPES = {"float64": "f64", "float32": "f32", "float16": "f16", "bfloat16": "bf16",
           "float8_e4m3fn": "e4m3", "int32": "i32", "int64": "i64"}
GATES = {None: 0, "silu": 1}
BLOCK = 128
MAX_EXPERTS = 1024


class DenseArg(ct.Structure):
    _fields_ = [("rows", ct.c_int64), ("cols", ct.c_int64), ("ld", ct.c_int64),
                ("data", ct.c_void_p), ("type", ct.c_int32), ("reserved", ct.c_int32)]


class RoutesArg(ct.Structure):
    _fields_ = [("tokens", ct.c_int64), ("top_k", ct.c_int32), ("reserved", ct.c_int32),
                ("pair_row", ct.c_void_p)]


class ScaledArg(ct.Structure):
    _fields_ = [("q", DenseArg), ("scale", ct.c_void_p), ("scale_ld", ct.c_int64)]


class BlocksArg(ct.Structure):
    _fields_ = [("groups", ct.c_int64), ("rows", ct.c_int64), ("cols", ct.c_int64),
                ("ld", ct.c_int64), ("group_stride", ct.c_int64), ("data", ct.c_void_p),
                ("scale", ct.c_void_p)]


_ready = None
_seen: dict = {}   # names of the dtypes seen


def _lib() -> ct.CDLL:
    global _ready
    if _ready is not None:
        return _ready
    lib = load()
    # structures are passed by their addresses, which _Call keeps alive: cheaper per call than byref
    vp, dev = ct.c_void_p, ct.c_int32
    dense = routes = scaled = blocks = vp
    sigs = {
        "appt_route": [dense, ct.c_int64, vp, vp, vp, vp, ct.c_size_t, dev, vp],
        "appt_dispatch": [routes, dense, vp, dense, dev, vp],
        "appt_combine": [routes, dense, vp, dense, dev, vp],
        "appt_combine_grad": [routes, dense, dense, vp, dense, vp, dev, vp],
        "appt_quantize": [dense, ct.c_int32, vp, scaled, dev, vp],
        "appt_dispatch_quantize": [routes, dense, scaled, dev, vp],
        "appt_scaled_product": [scaled, blocks, vp, dense, dev, vp],
    }
    for name, argtypes in sigs.items():
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = argtypes, ct.c_int
    lib.appt_route_workspace.argtypes = [ct.c_int64, ct.c_int32, ct.c_int64]
    lib.appt_route_workspace.restype = ct.c_size_t
    lib.appt_scaled_product_status.argtypes, lib.appt_scaled_product_status.restype = [dev], ct.c_int
    lib.appt_scaled_product_tile.argtypes = [ct.c_int64, ct.c_int64, ct.c_int64, ct.c_int32, vp, vp]
    lib.appt_scaled_product_tile.restype = ct.c_int
    lib.appt_scaled_product_give_up.argtypes = [ct.c_int32]
    lib.appt_scaled_product_give_up.restype = None
    _ready = lib
    return lib


class Dense:
    """An operand given by its device pointer: shape (any number of dimensions), strides in
    elements and a type of TYPES."""

    def __init__(self, ptr: int, shape: tuple, type: str, stride: tuple | None = None,
                 device: int = 0):
        if type not in TYPES:
            raise ApptError(f"unknown type {type!r}: one of {', '.join(TYPES)}")
        self.ptr, self.shape, self.type, self.device = int(ptr), tuple(map(int, shape)), type, device
        if stride is None:
            stride, n = [], 1
            for s in reversed(self.shape):
                stride.insert(0, n)
                n *= max(s, 1)
        self.strides = tuple(map(int, stride))
        if len(self.strides) != len(self.shape):
            raise ApptError("shape and stride differ in length")

    @staticmethod
    def of(t, name: str) -> "Dense":
        if isinstance(t, Dense):
            return t
        try:
            dtype, where = t.dtype, t.device
            d = Dense.__new__(Dense)
            d.ptr, d.shape, d.strides = t.data_ptr(), tuple(t.shape), t.stride()
            kind, d.device = where.type, where.index or 0
        except (AttributeError, TypeError):
            raise ApptError(f"{name}: needs a tensor on a CUDA device or a Dense") from None
        if kind != "cuda":
            raise ApptError(f"{name} is not on a CUDA device")
        if dtype not in _seen:
            _seen[dtype] = str(dtype).split(".")[-1]
        d.type = _DTYPES.get(_seen[dtype])
        if d.type is None:
            raise ApptError(f"{name}: type {_seen[dtype]} is not supported")
        return d


class _Call:
    """A library call with its arguments built once."""

    def __init__(self, entry: str):
        self._entry = entry
        self._fn = getattr(_lib(), entry)
        self._keep: list = []
        self._device: int | None = None

    def _dense(self, t, name: str, dims: int, types=None) -> Dense:
        d = Dense.of(t, name)
        if len(d.shape) != dims:
            raise ApptError(f"{name}: needs {dims} dimension{'s' if dims > 1 else ''}")
        if types is not None and d.type not in types:
            raise ApptError(f"{name}: needs type {' or '.join(types)}, not {d.type}")
        if self._device is None:
            self._device = d.device
        elif d.device != self._device:
            raise ApptError(f"{name} is on device {d.device}, other operands on {self._device}")
        if d.shape[-1] > 1 and d.strides[-1] != 1:
            raise ApptError(f"{name}: neighbouring columns must be neighbours in memory")
        self._keep.append(t)
        return d

    def _matrix(self, t, name: str, types=None) -> DenseArg:
        d = self._dense(t, name, 2, types)
        rows, cols = d.shape
        return DenseArg(rows, cols, d.strides[0] if rows > 1 else cols, d.ptr, TYPES[d.type], 0)

    def _flat(self, t, name: str, types, count: int | None = None, dims: int = 1) -> int | None:
        """The pointer of a contiguous array."""
        if t is None:
            return None
        d = self._dense(t, name, dims, types)
        n = 1
        for size, stride in zip(reversed(d.shape), reversed(d.strides)):
            if size > 1 and stride != n and 0 not in d.shape:
                raise ApptError(f"{name} must be contiguous")
            n *= size
        if count is not None and n != count:
            raise ApptError(f"{name}: needs {count} entries, not {n}")
        return d.ptr

    def _routes(self, r: "Routes") -> RoutesArg:
        if not isinstance(r, Routes):
            raise ApptError("routes: needs a Routes")
        # (ctypes would cut larger numbers to the field's width)
        if min(r.tokens, r.top_k) < 0 or max(r.tokens, r.top_k) >= 1 << 31:
            raise ApptError("routes: needs tokens >= 0, top_k >= 1 and tokens * top_k < 2^31 - 1")
        ptr = self._flat(r.pair_row, "pair_row", ("i32",), r.tokens * r.top_k)
        return RoutesArg(r.tokens, r.top_k, 0, ptr)

    def _weights(self, w, name: str, r: "Routes", type: int) -> int | None:
        if w is None:
            return None
        d = Dense.of(w, name)
        if d.shape != (r.tokens, r.top_k):
            raise ApptError(f"{name}: needs the shape ({r.tokens}, {r.top_k}), not {d.shape}")
        return self._flat(w, name, ("f64" if type == TYPES["f64"] else "f32",), dims=2)

    def _scaled(self, q, scale, name: str) -> ScaledArg:
        m = self._matrix(q, name, ("e4m3",))
        s = self._matrix(scale, f"{name}'s scale", ("f32",))
        need = (-(-m.cols // BLOCK), m.rows)
        if (s.rows, s.cols) != need:
            raise ApptError(f"{name}'s scale: needs the shape {need}, not {(s.rows, s.cols)}")
        return ScaledArg(m, s.data, s.ld)

    def _set(self, *args) -> None:
        self._structures = [a for a in args if isinstance(a, ct.Structure)]
        self._args = tuple(ct.addressof(a) if isinstance(a, ct.Structure) else a for a in args)
        self._args += (self._device,)

    def run(self, stream: int | None = None):
        """Makes the call on `stream`; returns self."""
        rc = self._fn(*self._args, stream)
        if rc:
            _check(rc, self._entry)
        return self


class Routes:
    """Where Route put each pair: pair_row has an int32 entry for each of the tokens * top_k
    pairs, its sorted row, -1 for a dropped pair. No two kept pairs have the same row."""

    def __init__(self, tokens: int, top_k: int, pair_row):
        self.tokens, self.top_k, self.pair_row = int(tokens), int(top_k), pair_row


def route_workspace_bytes(tokens: int, top_k: int, experts: int) -> int:
    """Bytes of device workspace for Route. Calls that may run at the same time need one each."""
    n = 0
    # (ctypes would cut larger numbers to the argument's width)
    if 0 <= min(tokens, top_k, experts) and max(tokens, top_k, experts) < 1 << 31:
        n = int(_lib().appt_route_workspace(tokens, top_k, experts))
    if n == 0:
        raise ApptError(f"no route of {tokens} x {top_k} pairs to {experts} experts: needs top_k "
                        f">= 1, 1 to {MAX_EXPERTS} experts and fewer than 2^31 - 1 pairs")
    return n


class Route(_Call):
    """Sorts the pairs of ids [tokens, top_k] (i32 or i64; an id outside [0, experts) drops its
    pair) by expert, stably: fills expert_ptr [experts + 1], row_pair and pair_row
    [tokens * top_k], all i32. workspace: a device buffer of route_workspace_bytes()."""

    def __init__(self, ids, experts: int, expert_ptr, row_pair, pair_row, workspace):
        super().__init__("appt_route")
        if not 1 <= experts <= MAX_EXPERTS:   # (ctypes would cut larger numbers)
            raise ApptError(f"experts must lie in [1, {MAX_EXPERTS}]")
        m = self._matrix(ids, "ids", ("i32", "i64"))
        pairs = m.rows * m.cols
        if isinstance(workspace, Dense):
            room = workspace.shape[0] if len(workspace.shape) == 1 else 0
            size = {"f64": 8, "i64": 8, "f32": 4, "i32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
            ptr, room = workspace.ptr, room * size[workspace.type]
        else:
            try:
                ptr, room = workspace.data_ptr(), workspace.numel() * workspace.element_size()
                if not workspace.is_contiguous():
                    raise ApptError("workspace must be contiguous")
            except AttributeError:
                raise ApptError("workspace: needs a tensor on a CUDA device or a Dense") from None
        self._keep.append(workspace)
        self._set(m, experts, self._flat(expert_ptr, "expert_ptr", ("i32",), experts + 1),
                  self._flat(row_pair, "row_pair", ("i32",), pairs),
                  self._flat(pair_row, "pair_row", ("i32",), pairs), ptr, room)


class Dispatch(_Call):
    """y[pair_row[p]] = weights[p] * x[p // top_k] for kept pairs (weights None: a copy). x has a
    row for each token, y the sorted rows; one type of f64, f32, f16, bf16; weights
    [tokens, top_k] f32 (f64 with f64 data). Gradients: of x Combine(routes, dy, dx, weights), of
    the weights CombineGrad(routes, x, dy, dweights=dw)."""

    def __init__(self, routes: Routes, x, y, weights=None):
        super().__init__("appt_dispatch")
        r, mx, my = self._routes(routes), self._matrix(x, "x"), self._matrix(y, "y")
        self._set(r, mx, self._weights(weights, "weights", routes, mx.type), my)


class Combine(_Call):
    """y[t] = sum over j of weights[t, j] * h[pair_row[t, j]]; a token without kept pairs gets
    zeros. Sums in f32 (f64 with f64 data)."""

    def __init__(self, routes: Routes, h, y, weights=None):
        super().__init__("appt_combine")
        r, mh, my = self._routes(routes), self._matrix(h, "h"), self._matrix(y, "y")
        self._set(r, mh, self._weights(weights, "weights", routes, mh.type), my)


class CombineGrad(_Call):
    """Gradient of Combine: dh[pair_row[p]] = weights[p] * dy[p // top_k], dweights[p] =
    <dy[p // top_k], h[pair_row[p]]>, 0 for dropped pairs. dh or dweights may be None (not
    wanted), h too where dweights is."""

    def __init__(self, routes: Routes, dy, h, weights=None, dh=None, dweights=None):
        super().__init__("appt_combine_grad")
        r, mdy = self._routes(routes), self._matrix(dy, "dy")
        mh = self._matrix(h, "h") if h is not None else None
        w = self._weights(weights, "weights", routes, mdy.type)
        mdh = self._matrix(dh, "dh") if dh is not None else None
        self._set(r, mdy, mh, w, mdh, self._weights(dweights, "dweights", routes, mdy.type))


class Quantize(_Call):
    """Rows of x to e4m3 with an f32 scale for each row and block of 128 columns: scale
    [ceil(cols / 128), rows], q [rows, cols]. gate "silu": the values are silu(x[:, :n]) * x[:, n:],
    in f32, silu taken as 0 below -87.3.
    rows_ptr (one i32 on the device): only that many rows are read and written."""

    def __init__(self, x, q, scale, rows_ptr=None, gate: str | None = None):
        super().__init__("appt_quantize")
        if gate not in GATES:
            raise ApptError(f"unknown gate {gate!r}")
        m = self._matrix(x, "x")
        self._set(m, GATES[gate], self._flat(rows_ptr, "rows_ptr", ("i32",), 1),
                  self._scaled(q, scale, "q"))


class DispatchQuantize(_Call):
    """Quantize of each token's row, written to its kept pairs' sorted rows."""

    def __init__(self, routes: Routes, x, q, scale):
        super().__init__("appt_dispatch_quantize")
        r, m = self._routes(routes), self._matrix(x, "x")
        self._set(r, m, self._scaled(q, scale, "q"))


class ScaledProduct(_Call):
    """y[r] = a[r] @ w[g].T for the rows r of group g, expert_ptr[g] .. expert_ptr[g + 1] - 1 (None
    with one group: all rows), in 8 bits: a [rows, k] e4m3 with a_scale [ceil(k / 128), rows], w
    [groups, n, k] (or [n, k]) e4m3 with w_scale [groups, ceil(n / 128), ceil(k / 128)], y
    [rows, n] f32, f16 or bf16. Rows of a and w start on 16 bytes. Sums in f32."""

    def __init__(self, a, a_scale, w, w_scale, y, expert_ptr=None):
        super().__init__("appt_scaled_product")
        ma = self._scaled(a, a_scale, "a")
        d = Dense.of(w, "w")
        dims = len(d.shape)
        if dims not in (2, 3):
            raise ApptError("w: needs 2 or 3 dimensions")
        d = self._dense(w, "w", dims, ("e4m3",))
        groups = d.shape[0] if dims == 3 else 1
        n, k = d.shape[-2:]
        ld = d.strides[-2] if n > 1 else -(-k // 16) * 16
        step = d.strides[0] if dims == 3 and groups > 1 else 0
        need = (groups, -(-n // BLOCK), -(-k // BLOCK))[3 - dims:]
        scale = self._dense(w_scale, "w_scale", dims, ("f32",))
        if scale.shape != need:   # blocks the other way round have as many entries
            raise ApptError(f"w_scale: needs the shape {need}, not {scale.shape}")
        sw = self._flat(w_scale, "w_scale", ("f32",), dims=dims)
        mw = BlocksArg(groups, n, k, ld, step, d.ptr, sw)
        ptr = self._flat(expert_ptr, "expert_ptr", ("i32",), groups + 1)
        self._set(ma, mw, ptr, self._matrix(y, "y"))


def product_tile(rows: int, n: int, groups: int = 1, sms: int = 148) -> tuple[int, int]:
    """Rows and columns of the tile of y that a ScaledProduct of these sizes goes by."""
    if not 0 <= min(rows, n, groups, sms) <= max(rows, n, groups, sms) < 1 << 31:   # (cut by ctypes)
        raise ApptError("no product has these sizes")
    out = (ct.c_int32 * 2)()
    _check(_lib().appt_scaled_product_tile(rows, n, groups, sms, ct.addressof(out),
                                           ct.addressof(out) + 4), "appt_scaled_product_tile")
    return out[0], out[1]


def check_products(device: int = 0) -> None:
    """Waits for the device and raises if a ScaledProduct on it has given up a wait since the last
    check (its y then holds NaN where it was not computed)."""
    _check(_lib().appt_scaled_product_status(device), "appt_scaled_product_status")


def make_products_give_up(on: bool) -> None:
    """For tests of what a program does when a product gives up a wait: those that run from now on
    do, in their first tiles."""
    _lib().appt_scaled_product_give_up(1 if on else 0)

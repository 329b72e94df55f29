"""Operators on rows of typed device tensors: the Python face of the entries of that section of include/skm_hip.h.

Rows of a table looked up by id and the table's gradient, rows sorted by the groups that a router chose and brought back
with weights, with their gradients, rows quantised to 8 bits and products of them.

Arguments are device tensors of whatever library the caller uses: anything with ``shape``, ``stride()``, ``dtype``,
``data_ptr()`` and, where it has one, ``device`` (a torch tensor), or a ``DeviceArray`` of this package.  Results go into
tensors that the caller passes, and are returned; nothing is copied, cast or allocated.  Calls are queued on the stream that
the object was made with.

    ops = RowOperators(device=0, stream=torch.cuda.current_stream().cuda_stream)
    ops.route(choices, n_groups, slots, offsets)
    ops.dispatch(x, slots, rows)
    ops.quantize(rows, q, scales)
    ops.product(q, scales, weights, weight_scales, products, offsets=offsets)
    ops.combine(products, slots, out, weights=shares)

Shapes, types, layouts and devices are checked on the host (ValueError, TypeError); indices are not, and one that points
outside of its table stands for no row.

The operators work on memory, beside torch's autograd: a tensor that requires gradients is taken like any other, no graph is
recorded, and a write into a tensor does not raise its version counter.  Gradients come from the calls named for them, for instance
in the ``backward`` of a ``torch.autograd.Function``.

torch's wheel carries a HIP runtime of its own, and the first one that a process loads has to serve both: import torch before
this package (tensors of a torch that came later are refused with a RuntimeError).
"""
import ctypes

import numpy as np

from . import _capi

def _dtype_name(dtype):
    """"float32" for numpy's and torch's float32 alike."""
    if isinstance(dtype, (np.dtype, type)):
        return np.dtype(dtype).name
    return str(dtype).rsplit(".", 1)[-1]


def _one_runtime():
    """Refuses tensors of a torch that came with a second HIP runtime: streams and memory of one mean nothing to the other."""
    with open("/proc/self/maps") as maps:
        found = {line.split(None, 5)[5].rstrip("\n") for line in maps if "/libamdhip64.so" in line}
    if len(found) > 1:
        raise RuntimeError(f"two HIP runtimes are loaded ({', '.join(sorted(found))}): import torch before superkmeans_amd")


class _Kinds(dict):
    """dtype object -> code of the C interface, for the types that an argument may have; filled as dtypes come along."""

    def __init__(self, codes):
        super().__init__()
        self.codes = codes

    def __missing__(self, dtype):
        if type(dtype).__module__.partition(".")[0] == "torch":
            _one_runtime()
        name = _dtype_name(dtype)
        if name not in self.codes:
            raise TypeError(f"must be {' or '.join(self.codes)}, not {name}")
        self[dtype] = self.codes[name]
        return self[dtype]


_VALUES = _Kinds({"float32": 0, "float16": 1, "bfloat16": 2})  # SKM_F32, SKM_F16, SKM_BF16
_IDS = _Kinds({"int32": 3, "uint32": 3, "int64": 4})  # SKM_U32 (a negative 32-bit id is a large one: no row), SKM_I64
_WORDS = _Kinds({"int32": 3, "uint32": 3})
_STEPS = _Kinds({"int8": 5})
_F32 = _Kinds({"float32": 0})
_SCRATCH = _Kinds({"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "uint32": 4, "int64": 8, "int8": 1, "uint8": 1})  # sizes
_SIGNED_ROWS = 1 << 31


class _Closed:
    """What an object has in the place of its context once it is closed."""

    handle = None


class RowOperators:
    """The operators on one device and stream.

    Parameters
    ----------
    device : int or None
        Device of every tensor that the calls get: 0, or the context's where one is given.
    stream : int or None
        Handle of the stream to queue on (0: the device's default stream); it has to outlive the object.  Give the stream that
        the tensors are made and used on: work on one stream runs in order, work on two does not.  None: a stream of the
        object's own.  Nothing makes that wait for work that the caller queued elsewhere, so wait for such work before a call, and
        ``sync`` before its results are used elsewhere or its tensors are released (the device's default stream and this one
        wait for each other by themselves; no other stream does).
    ctx : Context or None
        An existing context to work on instead; the object is of no use once that is closed.

    An object is not thread-safe: calls from several threads take an object each.
    """

    def __init__(self, device=None, stream=None, ctx=None):
        self.ctx = None
        self._owned = ctx is None
        if ctx is not None:
            has = getattr(ctx, "device", device)
            if device not in (None, has):
                raise ValueError(f"the context is on device {has}, not on device {device}")
            if stream is not None:
                raise ValueError("a context has its stream already")
            device = has
        self.device = 0 if device is None else device
        self.ctx = _capi.Context(self.device, stream) if ctx is None else ctx
        self._lib = self.ctx.lib
        self._context = self.ctx  # its handle is None once it is closed: the library refuses a null context


    def close(self):
        """Releases the context, if it is the object's own."""
        if self._owned and self.ctx is not None:
            self.ctx.close()
        self.ctx, self._context = None, _Closed

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def sync(self):
        """Waits for the stream."""
        self._call(self._lib.skm_sync(self._context.handle))

    # -- arguments ---------------------------------------------------------------------------------------------------
    # A decoding step's calls are short: these checks are written for few attribute reads, not for few lines.

    def _where(self, x, what):
        """The address of a tensor on this device."""
        try:
            index = x.get_device()
        except AttributeError:
            where = getattr(x, "device", None)
            index = self.device if where is None else where.index if getattr(where, "type", "cuda") == "cuda" else -1
        if index != self.device:
            raise ValueError(f"{what} is on {getattr(x, 'device', f'device {index}')}, not on device {self.device}")
        return x.data_ptr() or None

    def _refuse(self, x, what, error):
        """Says what is wrong with an argument whose attributes did not fit."""
        for name in ("shape", "stride", "dtype", "data_ptr"):
            if not hasattr(x, name):
                raise TypeError(f"{what} must be a device tensor, not {type(x).__name__}") from None
        if isinstance(error, TypeError):
            raise TypeError(f"{what} {error}") from None
        raise ValueError(f"{what} has {len(x.shape)} dimensions, which is not what it should have") from None

    def _matrix(self, x, what, kinds):
        """(address, type code, rows, columns, row stride): columns next to each other, rows any distance apart."""
        try:
            kind = kinds[x.dtype]
            rows, columns = x.shape
            row_stride, column_stride = x.stride()
        except (AttributeError, TypeError, ValueError) as e:
            self._refuse(x, what, e)
        if column_stride != 1 and columns > 1:
            raise ValueError(f"{what} must have its columns next to each other")
        if row_stride < columns:
            if rows > 1:
                raise ValueError(f"{what} has rows that overlap")
            row_stride = columns
        return self._where(x, what), kind, rows, columns, row_stride

    def _vector(self, x, what, kinds):
        """(address, type code, length) of a contiguous vector."""
        try:
            kind = kinds[x.dtype]
            (n,) = x.shape
            (stride,) = x.stride()
        except (AttributeError, TypeError, ValueError) as e:
            self._refuse(x, what, e)
        if stride != 1 and n > 1:
            raise ValueError(f"{what} must be contiguous")
        return self._where(x, what), kind, n

    def _dense(self, x, what, kinds):
        """(address, type code, rows, columns) of a contiguous matrix."""
        at, kind, rows, columns, row_stride = self._matrix(x, what, kinds)
        if row_stride != columns and rows > 1:
            raise ValueError(f"{what} must be contiguous")
        return at, kind, rows, columns

    def _scratch(self, scratch):
        if scratch is None:
            return None, 0
        if not hasattr(scratch, "dtype"):
            raise TypeError(f"scratch must be a device tensor, not {type(scratch).__name__}")
        at, size, n = self._vector(scratch, "scratch", _SCRATCH)
        return at, n * size

    def _call(self, rc):
        if rc == 0:
            return
        if rc == _capi.SKM_ERR_INVALID:
            raise ValueError(self._lib.skm_last_error().decode())
        _capi.check(rc)

    @staticmethod
    def _signed(ids, rows):
        """Negative 32-bit ids are read as large ones, which are rows of a table that long."""
        if _dtype_name(ids.dtype) == "int32":
            raise ValueError(f"ids of int32 cannot point into {rows} rows")

    @staticmethod
    def _misfit(what, has, wants):
        raise ValueError(f"{what} must have shape {wants}, not {has}")

    @staticmethod
    def _same_kind(what, has, wants):
        raise TypeError(f"{what} must have the type of {wants}")

    # -- lookup ------------------------------------------------------------------------------------------------------

    def lookup(self, table, ids, out, scale=1.0):
        """out[t] = scale * table[ids[t]], zeros where the id is no row.

        table : (rows, d) float32, float16 or bfloat16;  ids : (n,) int32 (up to 2^31 rows), uint32 or int64;  out : (n, d) of the
        table's type.
        """
        table_at, kind, rows, d, table_stride = self._matrix(table, "table", _VALUES)
        ids_at, ids_kind, n = self._vector(ids, "ids", _IDS)
        out_at, out_kind, out_rows, out_d, out_stride = self._matrix(out, "out", _VALUES)
        if out_kind != kind:
            self._same_kind("out", out_kind, "table")
        if out_rows != n or out_d != d:
            self._misfit("out", (out_rows, out_d), (n, d))
        if rows > _SIGNED_ROWS:
            self._signed(ids, rows)
        self._call(self._lib.skm_lookup_rows(self._context.handle, table_at, kind, rows, d, table_stride, ids_at, ids_kind, n,
                                             scale, out_at, out_stride))
        return out

    def lookup_grad(self, grad, ids, out, scale=1.0, accumulate=False, scratch=None):
        """out[v] = scale * (sum of grad[t] over the t with ids[t] == v): the gradient of `lookup` for its table.

        grad : (n, d);  ids : (n,) as in `lookup`;  out : (rows, d) of grad's type or float32.  With `accumulate` it is added to
        out, and rows that no id names are not touched; else those become zeros.  scratch : a one-dimensional
        tensor of at least `lookup_grad_scratch` bytes, or None for the context's workspace (not under graph capture).
        """
        grad_at, kind, n, d, grad_stride = self._matrix(grad, "grad", _VALUES)
        ids_at, ids_kind, n_ids = self._vector(ids, "ids", _IDS)
        out_at, out_kind, rows, out_d, out_stride = self._matrix(out, "out", _VALUES)
        if out_kind != kind and out_kind != 0:
            self._same_kind("out", out_kind, "grad, or float32")
        if n_ids != n:
            self._misfit("ids", (n_ids,), (n,))
        if out_d != d:
            self._misfit("out", (rows, out_d), (rows, d))
        if rows > _SIGNED_ROWS:
            self._signed(ids, rows)
        scratch_at, scratch_bytes = self._scratch(scratch)
        self._call(self._lib.skm_lookup_rows_grad(self._context.handle, grad_at, kind, grad_stride, ids_at, ids_kind, n, rows, d,
                                                  scale, out_at, out_kind, out_stride, 1 if accumulate else 0, scratch_at,
                                                  scratch_bytes))
        return out

    def lookup_grad_scratch(self, n, rows, d):
        """Bytes of scratch that `lookup_grad` needs for n tokens and a table of rows x d."""
        need = ctypes.c_size_t()
        self._call(self._lib.skm_lookup_rows_grad_scratch(n, rows, d, ctypes.byref(need)))
        return need.value

    # -- rows sorted by group and back -------------------------------------------------------------------------------

    def route(self, choices, groups, slots, offsets, order=None, scratch=None):
        """Places of the choices in the stable order by group.

        choices : (n, k) int32 or uint32 group numbers, anything outside [0, groups) being no group.  Results: slots (n, k), the
        place of every choice or -1 (0xffffffff); offsets (groups + 1,), the first place of every group and the number of places;
        order (n * k,), the choice t * k + j at every place, -1 behind the last one.  scratch: as in `lookup_grad`.
        """
        choices_at, _, n, k = self._dense(choices, "choices", _WORDS)
        slots_at, _, slots_n, slots_k = self._dense(slots, "slots", _WORDS)
        offsets_at, _, n_offsets = self._vector(offsets, "offsets", _WORDS)
        if slots_n != n or slots_k != k:
            self._misfit("slots", (slots_n, slots_k), (n, k))
        if n_offsets != groups + 1:
            self._misfit("offsets", (n_offsets,), (groups + 1,))
        order_at = None
        if order is not None:
            order_at, _, n_order = self._vector(order, "order", _WORDS)
            if n_order != n * k:
                self._misfit("order", (n_order,), (n * k,))
        scratch_at, scratch_bytes = self._scratch(scratch)
        self._call(self._lib.skm_route(self._context.handle, choices_at, n, k, groups, slots_at, order_at, offsets_at, scratch_at,
                                       scratch_bytes))
        return slots, offsets

    def route_scratch(self, n, choices, groups):
        """Bytes of scratch that `route` needs."""
        need = ctypes.c_size_t()
        self._call(self._lib.skm_route_scratch(n, choices, groups, ctypes.byref(need)))
        return need.value

    def dispatch(self, x, slots, out):
        """out[slots[t, j]] = x[t]; rows of out that are nobody's place stay as they are.

        x : (n, d);  slots : (n, k), distinct places as `route` makes them;  out : (places, d) of x's type.
        """
        x_at, kind, n, d, x_stride = self._matrix(x, "x", _VALUES)
        slots_at, _, slots_n, k = self._dense(slots, "slots", _WORDS)
        out_at, out_kind, out_rows, out_d, out_stride = self._matrix(out, "out", _VALUES)
        if out_kind != kind:
            self._same_kind("out", out_kind, "x")
        if slots_n != n:
            self._misfit("slots", (slots_n, k), (n, k))
        if out_d != d:
            self._misfit("out", (out_rows, out_d), (out_rows, d))
        self._call(self._lib.skm_dispatch_rows(self._context.handle, x_at, kind, n, d, x_stride, slots_at, k, out_at, out_rows,
                                               out_stride))
        return out

    def combine(self, rows, slots, out, weights=None):
        """out[t] = sum over j of weights[t, j] * rows[slots[t, j]]; without weights also the gradient of `dispatch`.

        rows : (places, d);  slots : (n, k);  weights : (n, k) float32, float16 or bfloat16;  out : (n, d) of the rows' type.
        """
        rows_at, kind, n_rows, d, rows_stride = self._matrix(rows, "rows", _VALUES)
        slots_at, _, n, k = self._dense(slots, "slots", _WORDS)
        out_at, out_kind, out_rows, out_d, out_stride = self._matrix(out, "out", _VALUES)
        if out_kind != kind:
            self._same_kind("out", out_kind, "rows")
        if out_rows != n or out_d != d:
            self._misfit("out", (out_rows, out_d), (n, d))
        weights_at, weights_kind = None, 0
        if weights is not None:
            weights_at, weights_kind, weights_n, weights_k = self._dense(weights, "weights", _VALUES)
            if weights_n != n or weights_k != k:
                self._misfit("weights", (weights_n, weights_k), (n, k))
        self._call(self._lib.skm_combine_rows(self._context.handle, rows_at, kind, n_rows, d, rows_stride, slots_at, n, k,
                                              weights_at, weights_kind, out_at, out_stride))
        return out

    def combine_grad(self, grad, rows, slots, weights, grad_rows, grad_weights):
        """Gradients of `combine`: grad_rows[slots[t, j]] = weights[t, j] * grad[t], grad_weights[t, j] = <grad[t], rows[slots[t, j]]>.

        grad : (n, d);  rows and grad_rows : (places, d) of its type;  grad_weights : (n, k) of the weights' type.  Either result may
        be None, and rows where grad_weights is; weights None stands for ones (grad_weights is then of any value type).
        """
        grad_at, kind, n, d, grad_stride = self._matrix(grad, "grad", _VALUES)
        slots_at, _, slots_n, k = self._dense(slots, "slots", _WORDS)
        if slots_n != n:
            self._misfit("slots", (slots_n, k), (n, k))
        rows_at, rows_stride, n_rows, out_at, out_stride = None, d, None, None, d
        if rows is not None:
            rows_at, rows_kind, n_rows, rows_d, rows_stride = self._matrix(rows, "rows", _VALUES)
            if rows_kind != kind:
                self._same_kind("rows", rows_kind, "grad")
            if rows_d != d:
                self._misfit("rows", (n_rows, rows_d), (n_rows, d))
        elif grad_weights is not None:
            raise ValueError("grad_weights needs the rows")
        if grad_rows is not None:
            out_at, out_kind, out_rows, out_d, out_stride = self._matrix(grad_rows, "grad_rows", _VALUES)
            if out_kind != kind:
                self._same_kind("grad_rows", out_kind, "grad")
            if out_d != d or n_rows not in (None, out_rows):
                self._misfit("grad_rows", (out_rows, out_d), (out_rows if n_rows is None else n_rows, d))
            n_rows = out_rows
        weights_at, weights_kind, grad_weights_at = None, 0, None
        if weights is not None:
            weights_at, weights_kind, weights_n, weights_k = self._dense(weights, "weights", _VALUES)
            if weights_n != n or weights_k != k:
                self._misfit("weights", (weights_n, weights_k), (n, k))
        if grad_weights is not None:
            grad_weights_at, out_kind, weights_n, weights_k = self._dense(grad_weights, "grad_weights", _VALUES)
            if weights is not None and out_kind != weights_kind:
                self._same_kind("grad_weights", out_kind, "weights")
            if weights_n != n or weights_k != k:
                self._misfit("grad_weights", (weights_n, weights_k), (n, k))
            weights_kind = out_kind
        if n_rows == 0 and grad_weights is None:
            return grad_rows, grad_weights  # no row to write, and a library may give a tensor of none no address
        self._call(self._lib.skm_combine_rows_grad(self._context.handle, grad_at, kind, n, d, grad_stride, rows_at, n_rows or 0,
                                                   rows_stride, slots_at, k, weights_at, weights_kind, out_at, out_stride,
                                                   grad_weights_at))
        return grad_rows, grad_weights

    # -- 8-bit rows --------------------------------------------------------------------------------------------------

    def quantize(self, x, q, scales):
        """q[t, i] = the whole number nearest to 127 x[t, i] / max|x[t]|, scales[t] = max|x[t]| / 127.

        x : (n, d);  q : (n, d) int8;  scales : (n,) float32.  A row with an infinity or NaN gets scale NaN.
        """
        x_at, kind, n, d, x_stride = self._matrix(x, "x", _VALUES)
        q_at, _, q_n, q_d, q_stride = self._matrix(q, "q", _STEPS)
        scales_at, _, n_scales = self._vector(scales, "scales", _F32)
        if q_n != n or q_d != d:
            self._misfit("q", (q_n, q_d), (n, d))
        if n_scales != n:
            self._misfit("scales", (n_scales,), (n,))
        self._call(self._lib.skm_quantize_rows(self._context.handle, x_at, kind, n, d, x_stride, q_at, q_stride, scales_at))
        return q, scales

    def product(self, a, a_scales, b, b_scales, out, bias=None, offsets=None):
        """out[i, j] = (sum over k of a[i, k] b[j, k]) * a_scales[i] * b_scales[j] + bias[j], the sum exact.

        a : (m, k) int8;  b : (n, k) int8;  a_scales (m,), b_scales and bias (n,) float32;  out : (m, n).  With offsets (groups + 1,),
        as `route` makes them, b is (groups, n, k) and b_scales and bias (groups, n): the rows [offsets[g], offsets[g + 1]) are
        multiplied with b[g], and rows of out that are in no group stay as they are.
        """
        a_at, _, m, k, a_stride = self._matrix(a, "a", _STEPS)
        out_at, out_kind, out_m, n, out_stride = self._matrix(out, "out", _VALUES)
        a_scales_at, _, n_scales = self._vector(a_scales, "a_scales", _F32)
        if n_scales != m:
            self._misfit("a_scales", (n_scales,), (m,))
        bias_at = offsets_at = None
        groups, group_stride = 1, 0
        if offsets is None:
            b_at, _, b_n, b_k, b_stride = self._matrix(b, "b", _STEPS)
            b_scales_at, _, scales_n = self._vector(b_scales, "b_scales", _F32)
            if bias is not None:
                bias_at, _, bias_n = self._vector(bias, "bias", _F32)
                if bias_n != n:
                    self._misfit("bias", (bias_n,), (n,))
        else:
            try:
                _STEPS[b.dtype]
                groups, b_n, b_k = b.shape
                group_stride, b_stride, column_stride = b.stride()
            except (AttributeError, TypeError, ValueError) as e:
                self._refuse(b, "b", e)
            b_at = self._where(b, "b")
            if column_stride != 1 and b_k > 1:
                raise ValueError("b must have its columns next to each other")
            if b_n == 1:
                b_stride = max(b_stride, b_k)
            if b_stride < b_k or groups > 1 and group_stride < (b_n - 1) * b_stride + b_k:
                raise ValueError("b has rows that overlap")
            if groups == 1:
                group_stride = 0
            offsets_at, _, n_offsets = self._vector(offsets, "offsets", _WORDS)
            if n_offsets != groups + 1:
                self._misfit("offsets", (n_offsets,), (groups + 1,))
            b_scales_at, _, scales_groups, scales_n = self._dense(b_scales, "b_scales", _F32)
            if scales_groups != groups:
                self._misfit("b_scales", (scales_groups, scales_n), (groups, n))
            if bias is not None:
                bias_at, _, bias_groups, bias_n = self._dense(bias, "bias", _F32)
                if bias_groups != groups or bias_n != n:
                    self._misfit("bias", (bias_groups, bias_n), (groups, n))
        if out_m != m or b_n != n or b_k != k or scales_n != n:
            raise ValueError(f"a {(m, k)}, b {(b_n, b_k)}, b_scales of {scales_n} and out {(out_m, n)} do not fit together")
        self._call(self._lib.skm_product_i8(self._context.handle, a_at, m, a_stride, a_scales_at, b_at, n, k, b_stride, b_scales_at,
                                            bias_at, groups, group_stride, offsets_at, out_at, out_kind, out_stride))
        return out

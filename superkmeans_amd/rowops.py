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
"""
import ctypes

import numpy as np

from . import _capi

_VALUES = {"float32": 0, "float16": 1, "bfloat16": 2}  # SKM_F32, SKM_F16, SKM_BF16
_IDS = {"int32": 3, "uint32": 3, "int64": 4}  # SKM_U32 (a negative 32-bit id is a large one: no row), SKM_I64
_WORDS = ("int32", "uint32")
_SIZES = {"float32": 4, "float16": 2, "bfloat16": 2, "int32": 4, "uint32": 4, "int64": 8, "int8": 1, "uint8": 1}

_dtype_names = {}


def _dtype_name(dtype):
    """"float32" for numpy's and torch's float32 alike."""
    name = _dtype_names.get(dtype)
    if name is None:
        if isinstance(dtype, (np.dtype, type)):
            name = np.dtype(dtype).name
        else:
            name = str(dtype).rsplit(".", 1)[-1]
        _dtype_names[dtype] = name
    return name


class RowOperators:
    """The operators on one device and stream.

    Parameters
    ----------
    device : int
        Device of every tensor that the calls get.
    stream : int or None
        Handle of the stream to queue on (0: the device's default stream); it has to outlive the object.  None: a stream of
        the object's own, which callers order with their work through ``sync``.
    ctx : Context or None
        An existing context to work on instead.

    An object is not thread-safe: calls from several threads take an object each.
    """

    def __init__(self, device=0, stream=None, ctx=None):
        self._owned = ctx is None
        self.ctx = _capi.Context(device, stream) if ctx is None else ctx
        self.device = device
        self._lib = self.ctx.lib

    def close(self):
        """Releases the context, if it is the object's own."""
        if self._owned and self.ctx is not None:
            self.ctx.close()
        self.ctx = None

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
        self.ctx.sync()

    # -- arguments ---------------------------------------------------------------------------------------------------

    def _tensor(self, x, what, dtypes, ndim):
        """(address, dtype name, shape, strides in elements) of a tensor on this device."""
        if isinstance(x, _capi.DeviceArray):
            shape, strides, address, step = x.shape, [], x.ptr, 1
            for size in reversed(shape):
                strides.insert(0, step)
                step *= size
        else:
            try:
                shape, strides, address = x.shape, x.stride(), x.data_ptr()
            except AttributeError:
                raise TypeError(f"{what} must be a device tensor, not {type(x).__name__}") from None
            where = getattr(x, "device", None)
            if where is not None:
                kind = getattr(where, "type", "cuda")
                if kind != "cuda" or where.index != self.device:
                    raise ValueError(f"{what} is on {where}, not on device {self.device}")
        name = _dtype_name(x.dtype)
        if name not in dtypes:
            raise TypeError(f"{what} must be {' or '.join(dtypes)}, not {name}")
        if len(shape) != ndim:
            raise ValueError(f"{what} must have {ndim} dimension{'s' if ndim > 1 else ''}, not {len(shape)}")
        return address or None, name, shape, strides

    def _matrix(self, x, what, dtypes):
        """(address, dtype name, rows, columns, row stride): columns next to each other, rows any distance apart."""
        address, name, (rows, columns), (row_stride, column_stride) = self._tensor(x, what, dtypes, 2)
        if columns > 1 and column_stride != 1:
            raise ValueError(f"{what} must have its columns next to each other")
        if rows > 1:
            if row_stride < columns:
                raise ValueError(f"{what} has rows that overlap")
        else:
            row_stride = columns
        return address, name, rows, columns, row_stride

    def _dense(self, x, what, dtypes, shape):
        """(address, dtype name) of a contiguous tensor of the given shape."""
        address, name, has, strides = self._tensor(x, what, dtypes, len(shape))
        if tuple(has) != shape:
            raise ValueError(f"{what} must have shape {shape}, not {tuple(has)}")
        step = 1
        for size, stride in zip(reversed(shape), reversed(strides)):
            if size > 1 and stride != step:
                raise ValueError(f"{what} must be contiguous")
            step *= size
        return address, name

    def _slots(self, slots):
        address, _, (n, choices), _ = self._tensor(slots, "slots", _WORDS, 2)
        self._dense(slots, "slots", _WORDS, (n, choices))
        return address, n, choices

    def _scratch(self, scratch):
        if scratch is None:
            return None, 0
        name = _dtype_name(scratch.dtype)
        if name not in _SIZES:
            raise TypeError(f"scratch cannot be of {name}")
        address, _, (n,), (stride,) = self._tensor(scratch, "scratch", (name,), 1)
        if n > 1 and stride != 1:
            raise ValueError("scratch must be contiguous")
        return address, n * _SIZES[name]

    def _call(self, rc):
        if rc == _capi.SKM_ERR_INVALID:
            raise ValueError(self._lib.skm_last_error().decode())
        if rc != 0:
            _capi.check(rc)

    # -- lookup ------------------------------------------------------------------------------------------------------

    def lookup(self, table, ids, out, scale=1.0):
        """out[t] = scale * table[ids[t]], zeros where the id is no row.

        table : (rows, d) float32, float16 or bfloat16;  ids : (n,) int32, uint32 or int64;  out : (n, d) of the table's type.
        """
        table_at, kind, rows, d, table_stride = self._matrix(table, "table", _VALUES)
        ids_at, ids_kind, (n,), (ids_stride,) = self._tensor(ids, "ids", _IDS, 1)
        out_at, _, out_rows, out_d, out_stride = self._matrix(out, "out", (kind,))
        if n > 1 and ids_stride != 1:
            raise ValueError("ids must be contiguous")
        if (out_rows, out_d) != (n, d):
            raise ValueError(f"out must have shape {(n, d)}, not {(out_rows, out_d)}")
        self._call(self._lib.skm_lookup_rows(self.ctx.handle, table_at, _VALUES[kind], rows, d, table_stride, ids_at, _IDS[ids_kind], n,
                                             scale, out_at, out_stride))
        return out

    def lookup_grad(self, grad, ids, out, scale=1.0, accumulate=False, scratch=None):
        """out[v] = scale * (sum of grad[t] over the t with ids[t] == v): the gradient of `lookup` for its table.

        grad : (n, d);  ids : (n,) as in `lookup`;  out : (rows, d) of grad's type or float32.  With `accumulate` it is added to
        out, and rows that no id names are not touched; else those become zeros.  scratch : a one-dimensional
        tensor of at least `lookup_grad_scratch` bytes, or None for the context's workspace (not under graph capture).
        """
        grad_at, kind, n, d, grad_stride = self._matrix(grad, "grad", _VALUES)
        ids_at, ids_kind, (n_ids,), (ids_stride,) = self._tensor(ids, "ids", _IDS, 1)
        out_at, out_kind, rows, out_d, out_stride = self._matrix(out, "out", (kind, "float32"))
        if n > 1 and ids_stride != 1:
            raise ValueError("ids must be contiguous")
        if n_ids != n:
            raise ValueError(f"ids must have shape {(n,)}, not {(n_ids,)}")
        if out_d != d:
            raise ValueError(f"out must have {d} columns, not {out_d}")
        scratch_at, scratch_bytes = self._scratch(scratch)
        self._call(self._lib.skm_lookup_rows_grad(self.ctx.handle, grad_at, _VALUES[kind], grad_stride, ids_at, _IDS[ids_kind], n, rows, d,
                                                  scale, out_at, _VALUES[out_kind], out_stride, 1 if accumulate else 0, scratch_at,
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
        choices_at, _, (n, k), _ = self._tensor(choices, "choices", _WORDS, 2)
        self._dense(choices, "choices", _WORDS, (n, k))
        slots_at, _ = self._dense(slots, "slots", _WORDS, (n, k))
        offsets_at, _ = self._dense(offsets, "offsets", _WORDS, (groups + 1,))
        order_at = None if order is None else self._dense(order, "order", _WORDS, (n * k,))[0]
        scratch_at, scratch_bytes = self._scratch(scratch)
        self._call(self._lib.skm_route(self.ctx.handle, choices_at, n, k, groups, slots_at, order_at, offsets_at, scratch_at,
                                       scratch_bytes))
        return slots, offsets

    def route_scratch(self, n, choices, groups):
        """Bytes of scratch that `route` needs."""
        need = ctypes.c_size_t()
        self._call(self._lib.skm_route_scratch(n, choices, groups, ctypes.byref(need)))
        return need.value

    def dispatch(self, x, slots, out):
        """out[slots[t, j]] = x[t]; rows of out that are nobody's place stay as they are.

        x : (n, d);  slots : (n, k);  out : (places, d) of x's type.
        """
        x_at, kind, n, d, x_stride = self._matrix(x, "x", _VALUES)
        slots_at, slots_n, k = self._slots(slots)
        out_at, _, out_rows, out_d, out_stride = self._matrix(out, "out", (kind,))
        if slots_n != n or out_d != d:
            raise ValueError(f"slots must have {n} rows and out {d} columns, not {slots_n} and {out_d}")
        self._call(self._lib.skm_dispatch_rows(self.ctx.handle, x_at, _VALUES[kind], n, d, x_stride, slots_at, k, out_at, out_rows,
                                               out_stride))
        return out

    def combine(self, rows, slots, out, weights=None):
        """out[t] = sum over j of weights[t, j] * rows[slots[t, j]]; without weights also the gradient of `dispatch`.

        rows : (places, d);  slots : (n, k);  weights : (n, k) float32, float16 or bfloat16;  out : (n, d) of the rows' type.
        """
        rows_at, kind, n_rows, d, rows_stride = self._matrix(rows, "rows", _VALUES)
        slots_at, n, k = self._slots(slots)
        out_at, _, out_rows, out_d, out_stride = self._matrix(out, "out", (kind,))
        if (out_rows, out_d) != (n, d):
            raise ValueError(f"out must have shape {(n, d)}, not {(out_rows, out_d)}")
        weights_at, weights_type = None, 0
        if weights is not None:
            weights_at, name = self._dense(weights, "weights", _VALUES, (n, k))
            weights_type = _VALUES[name]
        self._call(self._lib.skm_combine_rows(self.ctx.handle, rows_at, _VALUES[kind], n_rows, d, rows_stride, slots_at, n, k, weights_at,
                                              weights_type, out_at, out_stride))
        return out

    def combine_grad(self, grad, rows, slots, weights, grad_rows, grad_weights):
        """Gradients of `combine`: grad_rows[slots[t, j]] = weights[t, j] * grad[t], grad_weights[t, j] = <grad[t], rows[slots[t, j]]>.

        grad : (n, d);  rows and grad_rows : (places, d) of its type;  grad_weights : (n, k) of the weights' type.  Either result may
        be None, and rows where grad_weights is; weights None stands for ones (grad_weights is then of any value type).
        """
        grad_at, kind, n, d, grad_stride = self._matrix(grad, "grad", _VALUES)
        slots_at, slots_n, k = self._slots(slots)
        if slots_n != n:
            raise ValueError(f"slots must have {n} rows, not {slots_n}")
        rows_at, rows_stride, n_rows, out_at, out_stride = None, d, None, None, d
        if rows is not None:
            rows_at, _, n_rows, rows_d, rows_stride = self._matrix(rows, "rows", (kind,))
            if rows_d != d:
                raise ValueError(f"rows must have {d} columns, not {rows_d}")
        elif grad_weights is not None:
            raise ValueError("grad_weights needs the rows")
        if grad_rows is not None:
            out_at, _, out_rows, out_d, out_stride = self._matrix(grad_rows, "grad_rows", (kind,))
            if out_d != d or n_rows not in (None, out_rows):
                raise ValueError("grad_rows must have the shape of rows")
            n_rows = out_rows
        weights_at, weights_type, grad_weights_at = None, 0, None
        if weights is not None:
            weights_at, name = self._dense(weights, "weights", _VALUES, (n, k))
            weights_type = _VALUES[name]
        if grad_weights is not None:
            kinds = _VALUES if weights is None else (name,)
            grad_weights_at, name = self._dense(grad_weights, "grad_weights", kinds, (n, k))
            weights_type = _VALUES[name]
        self._call(self._lib.skm_combine_rows_grad(self.ctx.handle, grad_at, _VALUES[kind], n, d, grad_stride, rows_at, n_rows or 0,
                                                   rows_stride, slots_at, k, weights_at, weights_type, out_at, out_stride,
                                                   grad_weights_at))
        return grad_rows, grad_weights

    # -- 8-bit rows --------------------------------------------------------------------------------------------------

    def quantize(self, x, q, scales):
        """q[t, i] = the whole number nearest to 127 x[t, i] / max|x[t]|, scales[t] = max|x[t]| / 127.

        x : (n, d);  q : (n, d) int8;  scales : (n,) float32.  A row with an infinity or NaN gets scale NaN.
        """
        x_at, kind, n, d, x_stride = self._matrix(x, "x", _VALUES)
        q_at, _, q_n, q_d, q_stride = self._matrix(q, "q", ("int8",))
        if (q_n, q_d) != (n, d):
            raise ValueError(f"q must have shape {(n, d)}, not {(q_n, q_d)}")
        scales_at, _ = self._dense(scales, "scales", ("float32",), (n,))
        self._call(self._lib.skm_quantize_rows(self.ctx.handle, x_at, _VALUES[kind], n, d, x_stride, q_at, q_stride, scales_at))
        return q, scales

    def product(self, a, a_scales, b, b_scales, out, bias=None, offsets=None):
        """out[i, j] = (sum over k of a[i, k] b[j, k]) * a_scales[i] * b_scales[j] + bias[j], the sum exact.

        a : (m, k) int8;  b : (n, k) int8;  a_scales (m,), b_scales and bias (n,) float32;  out : (m, n).  With offsets (groups + 1,),
        as `route` makes them, b is (groups, n, k) and b_scales and bias (groups, n): the rows [offsets[g], offsets[g + 1]) are
        multiplied with b[g], and rows of out that are in no group stay as they are.
        """
        a_at, _, m, k, a_stride = self._matrix(a, "a", ("int8",))
        out_at, out_kind, out_m, n, out_stride = self._matrix(out, "out", _VALUES)
        if offsets is None:
            groups, group_stride, offsets_at = 1, 0, None
            b_at, _, b_n, b_k, b_stride = self._matrix(b, "b", ("int8",))
            per_column = (n,)
        else:
            b_at, _, (groups, b_n, b_k), (group_stride, b_stride, column_stride) = self._tensor(b, "b", ("int8",), 3)
            if b_k > 1 and column_stride != 1:
                raise ValueError("b must have its columns next to each other")
            if b_n == 1:
                b_stride = b_k
            if groups == 1:
                group_stride = 0
            if b_n > 1 and b_stride < b_k or groups > 1 and group_stride < (b_n - 1) * b_stride + b_k:
                raise ValueError("b has rows that overlap")
            offsets_at, _ = self._dense(offsets, "offsets", _WORDS, (groups + 1,))
            per_column = (groups, n)
        if out_m != m or b_n != n or b_k != k:
            raise ValueError(f"a {(m, k)}, b {(b_n, b_k)} and out {(out_m, n)} do not fit together")
        a_scales_at, _ = self._dense(a_scales, "a_scales", ("float32",), (m,))
        b_scales_at, _ = self._dense(b_scales, "b_scales", ("float32",), per_column)
        bias_at = None if bias is None else self._dense(bias, "bias", ("float32",), per_column)[0]
        self._call(self._lib.skm_product_i8(self.ctx.handle, a_at, m, a_stride, a_scales_at, b_at, n, k, b_stride, b_scales_at, bias_at,
                                            groups, group_stride, offsets_at, out_at, _VALUES[out_kind], out_stride))
        return out

"""What superkmeans_amd.rowops refuses before anything reaches a device (no GPU needed).

The tensors here have the attributes of device tensors and no memory; the context's library is a stand-in that records the
calls which would have been made.
"""
import pytest

from superkmeans_amd import rowops


class Device:
    def __init__(self, type="cuda", index=0):
        self.type, self.index = type, index

    def __str__(self):
        return f"{self.type}:{self.index}"


class Tensor:
    def __init__(self, shape, dtype="float32", stride=None, device=Device(), at=0x1000):
        self.shape, self.dtype, self.device, self._at = tuple(shape), f"torch.{dtype}", device, at
        if stride is None:
            stride, step = [], 1
            for size in reversed(self.shape):
                stride.insert(0, step)
                step *= max(size, 1)
        self._stride = tuple(stride)

    def stride(self):
        return self._stride

    def data_ptr(self):
        return self._at


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


class Context:
    def __init__(self):
        self.lib, self.handle = Library(), 1


@pytest.fixture
def ops():
    o = rowops.RowOperators(ctx=Context())
    yield o
    o.close()


T, I = Tensor, lambda shape, **kw: Tensor(shape, "int32", **kw)


def q8(shape, **kw):
    return Tensor(shape, "int8", **kw)


BAD = {
    "lookup out of another type": lambda o: o.lookup(T((9, 4)), I((3,)), T((3, 4), "bfloat16")),
    "lookup out of another shape": lambda o: o.lookup(T((9, 4)), I((3,)), T((4, 4))),
    "lookup table of an integer type": lambda o: o.lookup(I((9, 4)), I((3,)), I((3, 4))),
    "lookup ids of a float type": lambda o: o.lookup(T((9, 4)), T((3,)), T((3, 4))),
    "lookup ids of two dimensions": lambda o: o.lookup(T((9, 4)), I((3, 1)), T((3, 4))),
    "lookup ids with gaps": lambda o: o.lookup(T((9, 4)), I((3,), stride=(2,)), T((3, 4))),
    "lookup table by columns": lambda o: o.lookup(T((9, 4), stride=(1, 9)), I((3,)), T((3, 4))),
    "lookup table broadcast": lambda o: o.lookup(T((9, 4), stride=(0, 1)), I((3,)), T((3, 4))),
    "lookup out on the host": lambda o: o.lookup(T((9, 4)), I((3,)), T((3, 4), device=Device("cpu", None))),
    "lookup table on another device": lambda o: o.lookup(T((9, 4), device=Device("cuda", 1)), I((3,)), T((3, 4))),
    "lookup of a list": lambda o: o.lookup([[1.0]], I((3,)), T((3, 4))),
    "gradient with too few ids": lambda o: o.lookup_grad(T((3, 4)), I((2,)), T((9, 4))),
    "gradient into half precision": lambda o: o.lookup_grad(T((3, 4)), I((3,)), T((9, 4), "float16")),
    "gradient between half types": lambda o: o.lookup_grad(T((3, 4), "bfloat16"), I((3,)), T((9, 4), "float16")),
    "gradient of other columns": lambda o: o.lookup_grad(T((3, 4)), I((3,)), T((9, 5))),
    "gradient with a matrix of scratch": lambda o: o.lookup_grad(T((3, 4)), I((3,)), T((9, 4)), scratch=T((9, 9))),
    "gradient with a number for scratch": lambda o: o.lookup_grad(T((3, 4)), I((3,)), T((9, 4)), scratch=4096),
    "route of 64-bit choices": lambda o: o.route(Tensor((3, 2), "int64"), 4, I((3, 2)), I((5,))),
    "route slots of another shape": lambda o: o.route(I((3, 2)), 4, I((2, 3)), I((5,))),
    "route too few offsets": lambda o: o.route(I((3, 2)), 4, I((3, 2)), I((4,))),
    "route order of another length": lambda o: o.route(I((3, 2)), 4, I((3, 2)), I((5,)), order=I((5,))),
    "route choices with gaps": lambda o: o.route(I((3, 2), stride=(4, 1)), 4, I((3, 2)), I((5,))),
    "dispatch with other rows": lambda o: o.dispatch(T((3, 4)), I((2, 2)), T((6, 4))),
    "dispatch with other columns": lambda o: o.dispatch(T((3, 4)), I((3, 2)), T((6, 5))),
    "dispatch to another type": lambda o: o.dispatch(T((3, 4)), I((3, 2)), T((6, 4), "float16")),
    "dispatch with a vector of slots": lambda o: o.dispatch(T((3, 4)), I((3,)), T((6, 4))),
    "combine to another shape": lambda o: o.combine(T((6, 4)), I((3, 2)), T((6, 4))),
    "combine weights of another shape": lambda o: o.combine(T((6, 4)), I((3, 2)), T((3, 4)), weights=T((2, 3))),
    "combine weights of integers": lambda o: o.combine(T((6, 4)), I((3, 2)), T((3, 4)), weights=I((3, 2))),
    "combine gradient without rows": lambda o: o.combine_grad(T((3, 4)), None, I((3, 2)), T((3, 2)), T((6, 4)), T((3, 2))),
    "combine gradient of other rows": lambda o: o.combine_grad(T((3, 4)), T((6, 4)), I((3, 2)), T((3, 2)), T((5, 4)), T((3, 2))),
    "combine gradient of another weight type": lambda o: o.combine_grad(T((3, 4)), T((6, 4)), I((3, 2)), T((3, 2)), T((6, 4)),
                                                                      T((3, 2), "bfloat16")),
    "quantize to unsigned bytes": lambda o: o.quantize(T((3, 4)), Tensor((3, 4), "uint8"), T((3,))),
    "quantize to another shape": lambda o: o.quantize(T((3, 4)), q8((3, 5)), T((3,))),
    "quantize scales by column": lambda o: o.quantize(T((3, 4)), q8((3, 4)), T((4,))),
    "product of float rows": lambda o: o.product(T((3, 8)), T((3,)), q8((5, 8)), T((5,)), T((3, 5))),
    "product of other lengths": lambda o: o.product(q8((3, 8)), T((3,)), q8((5, 9)), T((5,)), T((3, 5))),
    "product with scales by k": lambda o: o.product(q8((3, 8)), T((8,)), q8((5, 8)), T((5,)), T((3, 5))),
    "product to integers": lambda o: o.product(q8((3, 8)), T((3,)), q8((5, 8)), T((5,)), I((3, 5))),
    "product groups without a dimension": lambda o: o.product(q8((3, 8)), T((3,)), q8((5, 8)), T((5,)), T((3, 5)), offsets=I((2,))),
    "product groups of other offsets": lambda o: o.product(q8((3, 8)), T((3,)), q8((2, 5, 8)), T((2, 5)), T((3, 5)), offsets=I((2,))),
    "product groups that overlap": lambda o: o.product(q8((3, 8)), T((3,)), q8((2, 5, 8), stride=(8, 8, 1)), T((2, 5)), T((3, 5)),
                                                       offsets=I((3,))),
    "product with rows that overlap": lambda o: o.product(q8((3, 8)), T((3,)), q8((1, 5, 8), stride=(40, 4, 1)), T((1, 5)), T((3, 5)),
                                                          offsets=I((2,))),
    "product with a bias for all groups": lambda o: o.product(q8((3, 8)), T((3,)), q8((2, 5, 8)), T((2, 5)), T((3, 5)), bias=T((5,)),
                                                              offsets=I((3,))),
}


@pytest.mark.parametrize("what", sorted(BAD))
def test_refused(ops, what):
    with pytest.raises((ValueError, TypeError)):
        BAD[what](ops)
    assert ops.ctx.lib.calls == []


def test_arguments_reach_the_library_in_the_header_s_order(ops):
    ops.lookup(T((9, 4), stride=(6, 1), at=0x10), Tensor((3,), "int64", at=0x20), T((3, 4), stride=(5, 1), at=0x30), scale=2.0)
    ops.product(q8((3, 8), at=0x10), T((3,), at=0x20), q8((2, 5, 8), stride=(60, 10, 1), at=0x30), T((2, 5), at=0x40),
                Tensor((3, 5), "float16", at=0x50), bias=T((2, 5), at=0x60), offsets=I((3,), at=0x70))
    ops.combine_grad(T((3, 4), at=0x10), T((6, 4), at=0x20), I((3, 2), at=0x30), T((3, 2), at=0x40), T((6, 4), at=0x50), None)
    assert ops.ctx.lib.calls == [
        ("skm_lookup_rows", (1, 0x10, 0, 9, 4, 6, 0x20, 4, 3, 2.0, 0x30, 5)),
        ("skm_product_i8", (1, 0x10, 3, 8, 0x20, 0x30, 5, 8, 10, 0x40, 0x60, 2, 60, 0x70, 0x50, 1, 5)),
        ("skm_combine_rows_grad", (1, 0x10, 0, 3, 4, 4, 0x20, 6, 4, 0x30, 2, 0x40, 0, 0x50, 4, None)),
    ]


def test_one_row_may_have_any_stride(ops):
    """A library may give a tensor of one row any row stride, and one of a single column any column stride."""
    ops.lookup(T((9, 4)), I((1,)), T((1, 4), stride=(0, 1)))
    ops.dispatch(T((3, 1), stride=(1, 7)), I((3, 2)), T((6, 1), stride=(1, 3)))
    assert len(ops.ctx.lib.calls) == 2


def test_scratch_sizes_need_no_device(capi):
    import ctypes

    lib = capi.load()
    need = ctypes.c_size_t()
    assert lib.skm_route_scratch(0, 2, 8, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.skm_route_scratch(64, 8, 64, ctypes.byref(need)) == 0 and need.value == 0  # one launch, no scratch
    sizes = []
    for n in (10000, 100000, 1000000):
        assert lib.skm_route_scratch(n, 2, 64, ctypes.byref(need)) == 0
        sizes.append(need.value)
    assert 0 < sizes[0] < sizes[1] < sizes[2] < 64 << 20
    assert lib.skm_route_scratch(1 << 20, 1 << 11, 8, ctypes.byref(need)) == capi.SKM_ERR_INVALID
    assert lib.skm_route_scratch(4, 2, 0, ctypes.byref(need)) == capi.SKM_ERR_INVALID
    assert lib.skm_lookup_rows_grad_scratch(100000, 65536, 64, ctypes.byref(need)) == 0 and need.value > 100000 * 4
    assert lib.skm_lookup_rows_grad_scratch(10, 10, 0, ctypes.byref(need)) == capi.SKM_ERR_INVALID


def test_null_context_is_refused(capi):
    lib = capi.load()
    assert lib.skm_lookup_rows(None, None, 0, 1, 1, 1, None, 3, 1, 1.0, None, 1) == capi.SKM_ERR_INVALID
    assert lib.skm_route(None, None, 1, 1, 1, None, None, None, None, 0) == capi.SKM_ERR_INVALID
    assert lib.skm_product_i8(None, None, 1, 1, None, None, 1, 1, 1, None, None, 0, 0, None, None, 0, 1) == capi.SKM_ERR_INVALID
    assert lib.skm_quantize_rows(None, None, 0, 1, 1, 1, None, 1, None) == capi.SKM_ERR_INVALID


# Every entry with its arguments apart: name -> (rows, pitch, width) in bytes, and the call for a set of addresses (of the scratch the
# first bytes, all of which the calls need).
N, D, K, ROWS = 6, 8, 3, 9
ENTRIES = {
    "skm_lookup_rows": (
        {"table": (ROWS, 40, 32), "ids": (1, 48, 48), "out": (N, 48, 32)}, {"out": ("table", "ids")},
        lambda f, h, a: f(h, a["table"], 0, ROWS, D, 10, a["ids"], 4, N, 1.0, a["out"], 12)),
    "skm_lookup_rows_grad": (
        {"grad": (3000, 40, 32), "ids": (1, 24000, 24000), "out": (ROWS, 48, 32), "scratch": (1, 4096, 4096)},
        {"out": ("grad", "ids", "scratch"), "scratch": ("grad", "ids")},
        lambda f, h, a: f(h, a["grad"], 0, 10, a["ids"], 4, 3000, ROWS, D, 1.0, a["out"], 0, 12, 0, a["scratch"], 1 << 20)),
    "skm_route": (
        {"choices": (1, 120000, 120000), "slots": (1, 120000, 120000), "order": (1, 120000, 120000), "offsets": (1, 20, 20), "scratch": (1, 4096, 4096)},
        {"slots": ("choices", "order", "offsets"), "order": ("choices", "offsets"), "offsets": ("choices",),
         "scratch": ("choices", "slots", "order", "offsets")},
        lambda f, h, a: f(h, a["choices"], 10000, 3, 4, a["slots"], a["order"], a["offsets"], a["scratch"], 1 << 20)),
    "skm_dispatch_rows": (
        {"x": (N, 40, 32), "slots": (1, 72, 72), "out": (18, 48, 32)}, {"out": ("x", "slots")},
        lambda f, h, a: f(h, a["x"], 0, N, D, 10, a["slots"], K, a["out"], 18, 12)),
    "skm_combine_rows": (
        {"rows": (18, 40, 32), "slots": (1, 72, 72), "weights": (1, 36, 36), "out": (N, 48, 32)}, {"out": ("rows", "slots", "weights")},
        lambda f, h, a: f(h, a["rows"], 0, 18, D, 10, a["slots"], N, K, a["weights"], 1, a["out"], 12)),
    "skm_combine_rows_grad": (
        {"grad": (N, 40, 32), "rows": (18, 40, 32), "slots": (1, 72, 72), "weights": (1, 72, 72), "grad_rows": (18, 48, 32),
         "grad_weights": (1, 72, 72)},
        {"grad_rows": ("grad", "rows", "slots", "weights", "grad_weights"), "grad_weights": ("grad", "rows", "slots", "weights")},
        lambda f, h, a: f(h, a["grad"], 0, N, D, 10, a["rows"], 18, 10, a["slots"], K, a["weights"], 0, a["grad_rows"], 12, a["grad_weights"])),
    "skm_quantize_rows": (
        {"x": (N, 40, 32), "q": (N, 12, 8), "scales": (1, 24, 24)}, {"q": ("x",), "scales": ("x", "q")},
        lambda f, h, a: f(h, a["x"], 0, N, D, 10, a["q"], 12, a["scales"])),
    "skm_product_i8": (
        {"a": (N, 12, 8), "a_scale": (1, 24, 24), "b": (1, 120, 120), "b_scale": (1, 40, 40), "bias": (1, 40, 40), "offsets": (1, 12, 12),
         "out": (N, 32, 20)},
        {"out": ("a", "a_scale", "b", "b_scale", "bias", "offsets")},
        lambda f, h, a: f(h, a["a"], N, 12, a["a_scale"], a["b"], 5, D, 12, a["b_scale"], a["bias"], 2, 60, a["offsets"], a["out"], 0, 8)),
}
PAIRS = [(entry, out, other) for entry, (_, pairs, _) in ENTRIES.items() for out, others in pairs.items() for other in others]


@pytest.fixture
def refusing(capi):
    """The library with memory that is no context: a call that is refused never looks at it, one that is not finds no device."""
    import ctypes

    lib = capi.load()
    if capi.device_count() > 0:
        pytest.skip("the addresses here are no memory: without a device only")
    memory = ctypes.create_string_buffer(1 << 16)
    return lib, ctypes.addressof(memory), memory


def apart(entry):
    return {name: (i + 1) << 32 for i, name in enumerate(ENTRIES[entry][0])}


@pytest.mark.parametrize("entry", sorted(ENTRIES))
def test_arguments_that_are_apart_are_not_refused(refusing, capi, entry):
    lib, handle, _ = refusing
    assert ENTRIES[entry][2](getattr(lib, entry), handle, apart(entry)) not in (0, capi.SKM_ERR_INVALID)


@pytest.mark.parametrize("entry,out,other", PAIRS)
def test_outputs_over_other_arguments_are_refused(refusing, capi, entry, out, other):
    lib, handle, _ = refusing
    shapes, _, call = ENTRIES[entry]
    at = apart(entry)
    (rows, pitch, width), (other_rows, other_pitch, other_width) = shapes[out], shapes[other]
    end = (other_rows - 1) * other_pitch + other_width
    for place in (at[other], at[other] + (end - 1) // 16 * 16):  # the same beginning, and the other's last bytes
        if rows == 1 and other_rows > 1 and place != at[other]:
            place = at[other] + (other_rows - 1) * other_pitch // 16 * 16
        assert call(getattr(lib, entry), handle, {**at, out: place}) == capi.SKM_ERR_INVALID, (entry, out, other)
        message = lib.skm_last_error().decode()
        assert "overlaps" in message and entry in message, message


def test_columns_of_one_buffer_are_apart(refusing, capi):
    """Rows that lie between each other's rows share no memory; one byte more and they do."""
    lib, handle, _ = refusing
    at = 1 << 32

    def dispatch(x, out, x_stride, out_stride, d, slots=1 << 40):
        return lib.skm_dispatch_rows(handle, x, 0, 50, d, x_stride, slots, 1, out, 50, out_stride)

    assert dispatch(at, at + 32, 16, 16, 8) != capi.SKM_ERR_INVALID
    assert dispatch(at + 32, at, 16, 16, 8) != capi.SKM_ERR_INVALID
    assert dispatch(at + 160, at, 16, 16, 8) != capi.SKM_ERR_INVALID  # 2.5 rows on
    assert dispatch(at, at + 32, 16, 16, 9) == capi.SKM_ERR_INVALID
    assert dispatch(at, at + 28, 16, 16, 8) == capi.SKM_ERR_INVALID
    assert dispatch(at, at + 32, 16, 17, 8) == capi.SKM_ERR_INVALID  # other pitches: their rows meet somewhere
    # vectors are apart from the whole range of a result's rows
    assert dispatch(1 << 33, at, 256, 256, 8, slots=at + 32) == capi.SKM_ERR_INVALID
    assert dispatch(1 << 33, at, 256, 256, 8, slots=at - 200) != capi.SKM_ERR_INVALID
    assert dispatch(1 << 33, at, 256, 256, 8, slots=at - 196) == capi.SKM_ERR_INVALID
    assert dispatch(1 << 33, at, 256, 256, 8, slots=at + 1024 * 49 + 32) != capi.SKM_ERR_INVALID
    # a single row between the rows of the result
    assert lib.skm_dispatch_rows(handle, at, 0, 1, 8, 16, 1 << 40, 1, at + 32, 50, 16) != capi.SKM_ERR_INVALID
    assert lib.skm_dispatch_rows(handle, at + 64 * 7, 0, 1, 8, 16, 1 << 40, 1, at + 32, 50, 16) != capi.SKM_ERR_INVALID
    assert lib.skm_dispatch_rows(handle, at + 64 * 7 + 4, 0, 1, 8, 16, 1 << 40, 1, at + 32, 50, 16) == capi.SKM_ERR_INVALID
    # distances that wrap
    assert dispatch(1 << 33, at, 16, 1 << 60, 8) == capi.SKM_ERR_INVALID


class ContextOfDevice(Context):
    def __init__(self, device):
        super().__init__()
        self.device = device


class Owned(Tensor):
    """An allocation that knows its context, and through it the device."""

    def __init__(self, ctx, *args, **kw):
        super().__init__(*args, **kw)
        self.ctx = ctx
        del self.device

    def get_device(self):
        return self.ctx.device


def test_tensors_are_compared_with_the_context_s_device():
    ctx, elsewhere = ContextOfDevice(1), ContextOfDevice(0)
    there, here = Device("cuda", 1), Device("cuda", 0)
    with rowops.RowOperators(ctx=ctx) as ops:
        assert ops.device == 1
        ops.lookup(T((9, 4), device=there), I((3,), device=there), T((3, 4), device=there))
        ops.lookup(Owned(ctx, (9, 4)), Owned(ctx, (3,), "int32"), Owned(ctx, (3, 4)))
        assert len(ctx.lib.calls) == 2
        for bad in (lambda: ops.lookup(T((9, 4), device=here), I((3,), device=there), T((3, 4), device=there)),
                    lambda: ops.lookup(Owned(elsewhere, (9, 4)), Owned(ctx, (3,), "int32"), Owned(ctx, (3, 4)))):
            with pytest.raises(ValueError, match="not on device 1"):
                bad()
        assert len(ctx.lib.calls) == 2
    with pytest.raises(ValueError, match="device 1, not on device 0"):
        rowops.RowOperators(device=0, ctx=ctx)
    with pytest.raises(ValueError, match="stream"):
        rowops.RowOperators(stream=7, ctx=ctx)
    assert rowops.RowOperators(device=1, ctx=ctx).device == 1


def test_device_of_no_context(capi):
    import ctypes

    device = ctypes.c_int(7)
    assert capi.load().skm_ctx_get_device(None, ctypes.byref(device)) == capi.SKM_ERR_INVALID


def test_a_closed_context_is_not_used_again(capi):
    """The handle of a context is taken for each call: a closed one has none, and the library refuses that."""
    ctx = Context()
    ops = rowops.RowOperators(ctx=ctx)
    ctx.handle = None  # what Context.close leaves
    ops.lookup(T((9, 4)), I((3,)), T((3, 4)))
    ops.sync()
    assert [args[0] for _, args in ctx.lib.calls] == [None, None]
    ctx.lib, ctx.handle = capi.load(), None
    for closed in (False, True):
        ops = rowops.RowOperators(ctx=ctx)
        if closed:
            ops.close()
        for call in (lambda: ops.lookup(T((9, 4)), I((3,)), T((3, 4))), ops.sync):
            with pytest.raises(ValueError, match="null context"):
                call()


IMPORTS = {
    "torch first": "import torch; from superkmeans_amd import _capi; _capi.load()",
    "torch later": "from superkmeans_amd import _capi; _capi.load(); import torch",
}


@pytest.mark.parametrize("order", sorted(IMPORTS))
def test_a_second_hip_runtime_is_refused(order):
    """In processes of their own: what is loaded stays loaded."""
    import os
    import subprocess
    import sys

    program = IMPORTS[order] + """
import sys
sys.path.insert(0, "tests")
from test_rowops_refusals import Context
from superkmeans_amd.rowops import RowOperators
runtimes = {line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line}
x = torch.zeros((2, 4))
try:
    RowOperators(ctx=Context()).dispatch(x, torch.zeros((2, 1), dtype=torch.int32), x)
except (ValueError, RuntimeError) as e:
    print(len(runtimes), type(e).__name__)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", program], cwd=root, capture_output=True, text=True, timeout=200)
    assert r.returncode == 0, r.stderr[-2000:]
    runtimes, error = r.stdout.split()[-2:]
    if order == "torch first":
        assert runtimes == "1"
    # host tensors: with one runtime they are refused for their device
    assert error == ("RuntimeError" if int(runtimes) > 1 else "ValueError")


def test_signed_ids_of_more_rows_than_they_can_name(ops):
    """-5 in 32 bits is read as 2^32 - 5, a row of a table that long."""
    many, most = (1 << 31) + 1, 1 << 31
    calls = [
        lambda rows, kind: ops.lookup(T((rows, 1)), Tensor((3,), kind), T((3, 1))),
        lambda rows, kind: ops.lookup_grad(T((3, 1)), Tensor((3,), kind), T((rows, 1))),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="int32"):
            call(many, "int32")
    assert ops.ctx.lib.calls == []
    for call in calls:
        call(many, "uint32")
        call(many, "int64")
        call(most, "int32")
    assert len(ops.ctx.lib.calls) == 3 * len(calls)


def test_calls_without_tokens_or_rows_may_have_no_memory(refusing, capi):
    """Libraries give tensors of no elements no address: nothing to do is no error."""
    lib, handle, _ = refusing

    class Real(Context):
        def __init__(self):
            self.lib, self.handle = lib, handle

    ops = rowops.RowOperators(ctx=Real())
    empty = lambda shape, kind="float32": Tensor(shape, kind, at=0)
    ops.lookup(T((9, 4)), empty((0,), "int64"), empty((0, 4)))
    ops.lookup_grad(empty((0, 4)), empty((0,), "int32"), empty((0, 4)))
    ops.lookup_grad(empty((0, 4)), empty((0,), "int32"), T((9, 4)), accumulate=True)
    ops.lookup_grad(T((3, 4)), I((3,)), empty((0, 4)))
    ops.dispatch(empty((0, 4)), empty((0, 2), "int32"), empty((0, 4)))
    ops.dispatch(T((3, 4)), I((3, 2)), empty((0, 4)))
    ops.combine(empty((0, 4)), empty((0, 2), "int32"), empty((0, 4)), weights=empty((0, 2)))
    ops.combine_grad(empty((0, 4)), empty((0, 4)), empty((0, 2), "int32"), empty((0, 2)), empty((0, 4)), empty((0, 2)))
    ops.combine_grad(empty((0, 4)), None, empty((0, 2), "int32"), None, empty((0, 4)), None)
    ops.combine_grad(empty((0, 4)), empty((0, 4)), empty((0, 2), "int32"), None, None, empty((0, 2)))
    ops.combine_grad(T((3, 4)), None, I((3, 2)), T((3, 2)), empty((0, 4)), None)
    ops.quantize(empty((0, 4)), empty((0, 4), "int8"), empty((0,)))
    ops.product(empty((0, 8), "int8"), empty((0,)), q8((5, 8)), T((5,)), empty((0, 5)))
    ops.product(empty((0, 8), "int8"), empty((0,)), q8((2, 5, 8)), T((2, 5)), empty((0, 5)), offsets=I((3,)))
    with pytest.raises(ValueError, match="no output"):
        ops.combine_grad(T((3, 4)), T((6, 4)), I((3, 2)), T((3, 2)), None, None)


def test_the_process_s_libraries_are_looked_at_once_per_type(ops, monkeypatch):
    """Not for every call: that takes about as long as a hundred of them."""
    looks = []
    monkeypatch.setattr(rowops, "_one_runtime", lambda: looks.append(1))

    class Type:
        def __init__(self, name):
            self.name = name

        def __str__(self):
            return f"torch.{self.name}"

    Type.__module__ = "torch"
    kinds = {name: Type(name) for name in ("float32", "int64", "uint8")}

    def tensor(shape, kind):
        t = Tensor(shape, kind)
        t.dtype = kinds[kind]
        return t

    for call in range(3):
        ops.lookup_grad(tensor((3, 4), "float32"), tensor((3,), "int64"), tensor((9, 4), "float32"), scratch=tensor((4096,), "uint8"))
        if call == 0:
            first = len(looks)
    assert 0 < first == len(looks)
    assert ops.ctx.lib.calls[-1][1][-1] == 4096
    with pytest.raises(TypeError, match="scratch"):
        ops.lookup_grad(T((3, 4)), I((3,)), T((9, 4)), scratch=Tensor((64,), "float64"))

"""ctypes binding of libkg_gfx950.so, the gfx950 C ABI declared in include/kg_gfx950.h.

The slot structure is byte-for-byte the reference's ``_CArgSlot``
(kernel_gen/execute_engine/runtime_args.py:217-237) and the marshalling follows
``_RuntimeArgSupport.marshal_slots_for_abi`` (runtime_args.py:590-664): memory slots carry
a data pointer, element shape and element strides; ``None`` is an absent memory slot
(data = NULL, shape (0,), stride (1,)); Python ints and floats become INT / FLOAT slots.
Memory arguments must be ROCm device tensors: the library refuses host pointers.

There is no CPU fallback: if the shared object is missing this module raises.
"""

from __future__ import annotations

import ctypes
import os
import struct
from array import array
from numbers import Integral, Real
from pathlib import Path
from typing import Any, Sequence

PACKAGE_DIR = Path(__file__).resolve().parent
LIBRARY_PATH = PACKAGE_DIR / "libkg_gfx950.so"

KG_ARG_MEMORY = 1
KG_ARG_INT = 2
KG_ARG_FLOAT = 3

DTYPE_CODES = {
    "float32": 1,
    "float64": 2,
    "int32": 3,
    "int64": 4,
    "float16": 5,
    "bfloat16": 6,
}
# of the serving entries alone: caches, and int8 codes
CACHE_DTYPE_CODES = {"int8": 7, "float8_e4m3fn": 8}

ENTRY_POINTS = (
    "kg_gfx950_matmul_entry",
    "kg_gfx950_conv2d_entry",
    "kg_gfx950_flash_attention_entry",
    "kg_gfx950_kv_cache_store_entry",
    "kg_gfx950_kv_cache_load_entry",
    "kg_gfx950_tree_attention_entry",
    "kg_gfx950_adapter_matmul_entry",
    "kg_gfx950_kv_cache_assign_entry",
    "kg_gfx950_kv_cache_release_entry",
    "kg_gfx950_quantize_rows_entry",
    "kg_gfx950_int8_matmul_entry",
    "kg_gfx950_head_norm_rotate_entry",
)
CONTROL_SYMBOLS = (
    "kg_gfx950_set_launch_mode",
    "kg_gfx950_last_error",
    "kg_gfx950_abi_version",
    "kg_gfx950_cost",
    "kg_gfx950_fail",
    "kg_gfx950_check_memory_slot",
    "kg_gfx950_launch_stream",
    "kg_gfx950_launch_synchronous",
    "kg_gfx950_finish_launch",
)

# kg_gfx950_cost: op codes (KG_OP_*) and the order of its output array (KG_COST_*).
COST_OPS = {"matmul": 1, "conv2d": 2, "flash_attention": 3, "adapter_matmul": 4, "int8_matmul": 5}
COST_KINDS = ("MAC", "MFMA", "HBM_READ", "HBM_WRITE", "MFMA_CYCLES")


class KgArgSlot(ctypes.Structure):
    """C slot, identical in layout to the reference's ``_CArgSlot``."""

    _fields_ = [
        ("kind", ctypes.c_int),
        ("data", ctypes.c_void_p),
        ("shape", ctypes.POINTER(ctypes.c_longlong)),
        ("stride", ctypes.POINTER(ctypes.c_longlong)),
        ("rank", ctypes.c_ulonglong),
        ("dtype_code", ctypes.c_int),
        ("int_value", ctypes.c_longlong),
        ("float_value", ctypes.c_double),
    ]


class NativeLibraryError(RuntimeError):
    """libkg_gfx950.so is missing or an entry point returned non-zero."""

    def __init__(self, message: str, status: int = 0) -> None:
        super().__init__(message)
        self.status = status


_LIBRARY: ctypes.CDLL | None = None
# the entries taking the slots' address as an integer (call_entry packs them itself)
_ADDRESS_CALLS: dict[str, Any] = {}
# the entries' own addresses, and the host module that packs torch tensors into slots (None: not built, or no torch)
_ENTRY_ADDRESSES: dict[str, int] = {}
_FAST_CALL: Any = None


def library_path() -> Path:
    override = os.environ.get("KG_GFX950_LIBRARY")
    return Path(override) if override else LIBRARY_PATH


def load_library() -> ctypes.CDLL:
    """Load (once) and return the gfx950 library; raise if it has not been built."""

    global _LIBRARY, _FAST_CALL
    if _LIBRARY is not None:
        return _LIBRARY
    path = library_path()
    if not path.is_file():
        raise NativeLibraryError(
            f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'`"
        )
    # torch ships its own libamdhip64.so.7. Loaded first, it serves this library too (same
    # soname); loaded after this library, it would be a second HIP runtime in the process,
    # and device memory or kernels of one are not valid in the other.
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    lib = ctypes.CDLL(str(path))
    for name in ENTRY_POINTS:
        fn = getattr(lib, name)
        fn.argtypes = [ctypes.POINTER(KgArgSlot), ctypes.c_ulonglong]
        fn.restype = ctypes.c_int
        by_address = lib[name]  # a function object of its own, with its own argument types
        by_address.argtypes = [ctypes.c_void_p, ctypes.c_ulonglong]
        by_address.restype = ctypes.c_int
        _ADDRESS_CALLS[name] = by_address
        _ENTRY_ADDRESSES[name] = ctypes.cast(fn, ctypes.c_void_p).value
    lib.kg_gfx950_set_launch_mode.argtypes = [ctypes.c_int, ctypes.c_void_p]
    lib.kg_gfx950_set_launch_mode.restype = ctypes.c_int
    lib.kg_gfx950_last_error.argtypes = []
    lib.kg_gfx950_last_error.restype = ctypes.c_char_p
    lib.kg_gfx950_abi_version.argtypes = []
    lib.kg_gfx950_abi_version.restype = ctypes.c_int
    lib.kg_gfx950_cost.argtypes = [ctypes.c_int, ctypes.POINTER(KgArgSlot), ctypes.c_ulonglong,
                                   ctypes.POINTER(ctypes.c_longlong)]
    lib.kg_gfx950_cost.restype = ctypes.c_int
    try:
        from kernelcode_generate_amd import _kg_call

        _FAST_CALL = _kg_call.call
    except ImportError:  # (not built, built against another torch or Python, or no torch: the slots are packed here)
        _FAST_CALL = None
    _LIBRARY = lib
    return lib


class TensorSpec:
    """Shape, element strides and dtype of an operand, for cost queries without memory.

    ``data_ptr()`` returns a non-zero placeholder: a present memory slot needs a non-NULL
    pointer, and kg_gfx950_cost never dereferences it.
    """

    def __init__(self, shape: Sequence[int], dtype: str, strides: Sequence[int] | None = None) -> None:
        self.shape = tuple(int(d) for d in shape)
        self.dtype = str(dtype).replace("torch.", "")
        if strides is None:
            strides, step = [], 1
            for d in reversed(self.shape):
                strides.insert(0, step)
                step *= max(d, 1)
        self._strides = tuple(int(s) for s in strides)

    @classmethod
    def of(cls, value: Any) -> "TensorSpec":
        """Spec of a torch tensor or numpy array (numpy byte strides become element strides)."""

        if hasattr(value, "stride") and callable(value.stride):
            return cls(value.shape, str(value.dtype), value.stride())
        itemsize = int(value.itemsize)
        return cls(value.shape, value.dtype.name, [s // itemsize for s in value.strides])

    def stride(self) -> tuple[int, ...]:
        return self._strides

    def data_ptr(self) -> int:
        return 256


_DTYPE_CODE_OF: dict[Any, int] = {}  # dtype object (torch.dtype, numpy dtype or name) -> slot code


def dtype_code_of(value: Any) -> int:
    dtype = getattr(value, "dtype", "")
    code = _DTYPE_CODE_OF.get(dtype)
    if code is None:
        name = str(dtype).replace("torch.", "")
        code = DTYPE_CODES.get(name) or CACHE_DTYPE_CODES.get(name)
        if code is None:
            raise NativeLibraryError(f"unsupported memory dtype {name!r}", -1)
        _DTYPE_CODE_OF[dtype] = code
    return code


_MEMORY_KINDS: set[type] = set()  # classes whose objects are memory arguments (looked up once: a shape is made by asking)


def _is_memory(value: Any) -> bool:
    if type(value) in _MEMORY_KINDS:
        return True
    names = ("data_ptr", "shape", "stride", "dtype")
    if all(hasattr(type(value), name) for name in names):  # of the class: every object of it has them
        _MEMORY_KINDS.add(type(value))
        return True
    return all(hasattr(value, name) for name in names[:3])


# A KgArgSlot is eight 64-bit words (the 32-bit fields are padded to one each), so a call's
# slots, followed by the memory slots' shapes and strides, are packed as one array of int64: a
# ctypes structure and two ctypes arrays per slot took 8 us of a 12 us fp32 256^3 matmul call.
_SLOT_WORDS = ctypes.sizeof(KgArgSlot) // 8
_INT64 = 1 << 63
_pack_double = struct.Struct("d").pack
_unpack_int64 = struct.Struct("q").unpack


def _float_bits(value: float) -> int:
    return _unpack_int64(_pack_double(value))[0]


def _slot_words(args: Sequence[Any], address: int) -> list[int]:
    """The words of ``args`` (tensors / None / int / float), to lie at ``address``."""

    words: list[int] = []
    tail: list[int] = []  # shapes and strides of the memory slots
    at = address + 8 * _SLOT_WORDS * max(len(args), 1)  # of the next ones
    for position, arg in enumerate(args):
        kind = type(arg)
        if arg is None:
            words += (KG_ARG_MEMORY, 0, at, at + 8, 1, 0, 0, 0)
            tail += (0, 1)
            at += 16
        elif kind is int:
            words += (KG_ARG_INT, 0, 0, 0, 0, 0, arg, 0)
        elif kind is float:
            words += (KG_ARG_FLOAT, 0, 0, 0, 0, 0, 0, _float_bits(arg))
        elif kind in _MEMORY_KINDS or _is_memory(arg):  # (no number has a data_ptr)
            dims = arg.shape
            rank = len(dims)
            code = _DTYPE_CODE_OF.get(arg.dtype) or dtype_code_of(arg)
            words += (KG_ARG_MEMORY, arg.data_ptr(), at, at + 8 * (rank or 1), rank, code, 0, 0)
            if rank:
                tail += dims
                tail += arg.stride()
                at += 16 * rank
            else:
                tail += (0, 0)
                at += 16
        elif isinstance(arg, bool):
            raise NativeLibraryError(f"bool runtime arg at position {position} is not supported", -1)
        elif isinstance(arg, Integral):
            words += (KG_ARG_INT, 0, 0, 0, 0, 0, int(arg), 0)
        elif isinstance(arg, Real):
            words += (KG_ARG_FLOAT, 0, 0, 0, 0, 0, 0, _float_bits(float(arg)))
        else:
            raise NativeLibraryError(f"unsupported runtime arg at position {position}: {type(arg).__name__}", -1)
    if not words:
        words = [0] * _SLOT_WORDS
    words += tail
    return words


def _put_words(words: list[int], to: array) -> None:
    pack = _PACKERS.get(len(words))
    if pack is None:
        pack = _PACKERS[len(words)] = struct.Struct(f"{len(words)}q").pack_into
    try:
        pack(to, 0, *words)
    except struct.error:  # an integer beyond a C long long: its low 64 bits
        pack(to, 0, *((w + _INT64) % (2 * _INT64) - _INT64 for w in words))


_PACKERS: dict[int, Any] = {}  # number of words -> their packing


# Memory for the words of a call, and its address, while no call uses it. Taken and given back by a list's own pop and
# append, so that calls of two threads, or of a signal handler amid another, never have the same.
_CALL_WORDS = 512
_FREE_WORDS: list[tuple[array, int]] = []


def _take_words() -> tuple[array, int]:
    try:
        return _FREE_WORDS.pop()
    except IndexError:
        packed = array("q", bytes(8 * _CALL_WORDS))
        return packed, packed.buffer_info()[0]


def marshal_slots(args: Sequence[Any]) -> tuple[ctypes.Array, list[Any]]:
    """Build the C slot array for ``args`` (tensors / None / int / float)."""

    packed = array("q", bytes(8 * len(_slot_words(args, 0))))
    _put_words(_slot_words(args, packed.buffer_info()[0]), packed)
    slots = (KgArgSlot * max(len(args), 1)).from_buffer(packed)
    return slots, [packed, slots, *args]


def call_entry(entry_point: str, args: Sequence[Any], *, check: bool = True) -> int:
    """Invoke one gfx950 entry point with reference-ordered args; raise on non-zero if check."""

    lib = _LIBRARY or load_library()
    status = None
    if _FAST_CALL is not None and type(args) is tuple:
        address = _ENTRY_ADDRESSES.get(entry_point)
        if address is not None:
            status = _FAST_CALL(address, args)
    if status is None:
        status = _packed_call(lib, entry_point, args)
    if check and status != 0:
        detail = lib.kg_gfx950_last_error().decode("utf-8", "replace")
        raise NativeLibraryError(f"{entry_point} returned {status}: {detail}", status)
    return status


def _packed_call(lib: ctypes.CDLL, entry_point: str, args: Sequence[Any]) -> int:
    fn = _ADDRESS_CALLS.get(entry_point)
    own = _take_words()
    try:
        words = _slot_words(args, own[1])
        if fn is not None and len(words) <= _CALL_WORDS:
            _put_words(words, own[0])
            return fn(own[1], len(args))
        slots, keepalive = marshal_slots(args)
        status = int(getattr(lib, entry_point)(slots, ctypes.c_ulonglong(len(args))))
        del keepalive
        return status
    finally:
        _FREE_WORDS.append(own)


def cost(family: str, args: Sequence[Any]) -> dict[str, int]:
    """Per-call cost of ``family``'s entry on ``args`` (its full slot list; memory args may
    be TensorSpec), computed by kg_gfx950_cost without touching a GPU."""

    lib = load_library()
    op = COST_OPS.get(family)
    if op is None:
        raise NativeLibraryError(f"no cost model for {family!r}", -1)
    array, keepalive = marshal_slots(args)
    values = (ctypes.c_longlong * len(COST_KINDS))()
    status = int(lib.kg_gfx950_cost(op, array, ctypes.c_ulonglong(len(args)), values))
    del keepalive
    if status != 0:
        detail = lib.kg_gfx950_last_error().decode("utf-8", "replace")
        raise NativeLibraryError(f"kg_gfx950_cost({family}) returned {status}: {detail}", status)
    return {kind: int(values[i]) for i, kind in enumerate(COST_KINDS)}


def last_error() -> str:
    return load_library().kg_gfx950_last_error().decode("utf-8", "replace")


def set_launch_mode(synchronous: bool, stream: int | None = None) -> None:
    """synchronous=True: each entry waits for its kernel. False: enqueue on ``stream``."""

    load_library().kg_gfx950_set_launch_mode(1 if synchronous else 0, ctypes.c_void_p(stream or 0))


def matmul(out, lhs, rhs, bias=None, *tiles: int) -> None:
    call_entry("kg_gfx950_matmul_entry", (out, lhs, rhs, bias, *tiles))


def conv2d(out, x, weight, bias, stride=(1, 1), dilation=(1, 1), padding=(0, 0, 0, 0), tiles=(),
           memory_stage: int | None = None) -> None:
    """padding = (top, bottom, left, right); memory_stage: the LDS stage count (with 5 tiles)."""

    if memory_stage is not None and len(tiles) != 5:
        tiles = (1, 1, 1, 1, 1)
    stage = () if memory_stage is None else (int(memory_stage),)
    call_entry("kg_gfx950_conv2d_entry", (out, x, weight, bias, *stride, *dilation, *padding, *tiles, *stage))


def flash_attention(out, q, k, v, br: int = 64, bc: int = 64, scale: float = 1.0, causal: bool = False,
                    memory_stage: int | None = None) -> None:
    """memory_stage: the K/V ring depth of the MFMA kernel (2, 3 or 4)."""

    stage = () if memory_stage is None else (int(memory_stage),)
    call_entry("kg_gfx950_flash_attention_entry",
               (out, q, k, v, int(br), int(bc), float(scale), int(bool(causal)), *stage))


def kv_cache_store(k_cache, v_cache, k_scale, v_scale, k, v, slots) -> None:
    """Write rows k, v [T, heads, D] to the slots (int64 [T], page * page_size + offset; -1: none) of
    caches [pages, heads, page_size, D]; 8-bit ones (int8, float8_e4m3fn) with scales [pages, heads,
    page_size] (float32), others with None. No two tokens may name one slot."""

    call_entry("kg_gfx950_kv_cache_store_entry", (k_cache, v_cache, k_scale, v_scale, k, v, slots))


def kv_cache_load(k_out, v_out, k_cache, v_cache, k_scale, v_scale, page_table, lengths) -> None:
    """Read the first lengths[b] (int32 [B]) rows of each sequence back into k_out, v_out [B, heads, S, D],
    by its pages page_table[b] (int32 [B, P]). Rows past them are left as they are."""

    call_entry("kg_gfx950_kv_cache_load_entry", (k_out, v_out, k_cache, v_cache, k_scale, v_scale, page_table, lengths))


def tree_attention(out, q, k_cache, v_cache, k_scale, v_scale, page_table, context_lens, starts, mask=None,
                   scale: float = 1.0) -> None:
    """Attention of the tokens q [T, Hq, D] over the cache. Request b has tokens starts[b] to
    starts[b + 1] - 1 (int32 [B + 1]), whose own keys and values lie behind its context_lens[b] cached ones.
    Token j sees the context and the request's drafted tokens i with bit i % 64 of mask[starts[b] + j, i / 64]
    (int64 [T, W]); without a mask i <= j: a decoding step, a chain of drafts, a piece of a prompt."""

    call_entry("kg_gfx950_tree_attention_entry",
               (out, q, k_cache, v_cache, k_scale, v_scale, page_table, context_lens, starts, mask, float(scale)))


def adapter_matmul(out, x, weight, bias, a, b, index, scale=None) -> None:
    """out = x @ weight + bias, plus scale[l] * (x[m] @ a[l]) @ b[l] in each row m whose l = index[m]
    (int32 [M]) is an adapter (a [L, K, R], b [L, R, N]; scale: float32 [L], 1 where None)."""

    call_entry("kg_gfx950_adapter_matmul_entry", (out, x, weight, bias, a, b, index, scale))


def kv_cache_assign(slots, positions, starts, page_table, free_pages, free_count, context_lens, new_lens, page_size: int) -> None:
    """Pages and slots of new_lens[b] new tokens behind each request's context_lens[b] cached ones (int32 [B]): starts
    (int32 [B + 1]) of the requests' rows in the batch, and of each row its position (int32 [T]) and slot (int64 [T]), -1 behind the last.
    New pages come off the stack free_pages (int32 [F], free_count (int32 [1]) of them) and are entered in page_table (int32 [B, P])."""

    call_entry("kg_gfx950_kv_cache_assign_entry", (slots, positions, starts, page_table, free_pages, free_count, context_lens,
                                                   new_lens, int(page_size)))


def kv_cache_release(page_table, free_pages, free_count, keep_lens, held_lens, page_size: int) -> None:
    """Put the pages that request b's first keep_lens[b] tokens do not need, of those for held_lens[b], back on the stack:
    a request that ended (keep 0), drafted tokens that were rejected."""

    call_entry("kg_gfx950_kv_cache_release_entry", (page_table, free_pages, free_count, keep_lens, held_lens, int(page_size)))


def quantize_rows(codes, scale, x) -> None:
    """Rows x [M, K] as int8 codes [M, K] and float32 scales [M]: scale = max|x| / 127, code = x / scale rounded to nearest."""

    call_entry("kg_gfx950_quantize_rows_entry", (codes, scale, x))


def int8_matmul(out, x, x_scale, weight, w_scale, bias=None) -> None:
    """out = (x @ weight.T) * x_scale[:, None] * w_scale + bias, weight int8 [N, K], w_scale float32 [N]. x: int8 [M, K] with x_scale
    (float32 [M]), or of out's type with None: its rows are then quantised as by quantize_rows."""

    call_entry("kg_gfx950_int8_matmul_entry", (out, x, x_scale, weight, w_scale, bias))


def head_norm_rotate(q_out, k_out, q, k, q_weight, k_weight, cos, sin, positions, eps: float = 1e-6, neighbours: bool = False) -> None:
    """Norms over the heads of q [T, Hq, D] and k [T, Hk, D] (a side whose weight [D] is None: none), then the rotation of
    the pairs (i, i + R), or (2 i, 2 i + 1) of neighbours, by row positions[t] of cos and sin (float32 [S, R]). Tokens with positions
    outside the table (-1) are left as they are. The outputs may be the inputs."""

    call_entry("kg_gfx950_head_norm_rotate_entry", (q_out, k_out, q, k, q_weight, k_weight, cos, sin, positions, float(eps),
                                                    int(bool(neighbours))))

"""DLPack structs (restated from the public DLPack specification) and the
conversion of Python array objects into `DLTensor*` arguments for libkvcache.

Accepted inputs: this package's DeviceArray and HostBuffer (descriptors built
directly, no capsule), or any object implementing the DLPack protocol
(`__dlpack__`, e.g. a CUDA torch tensor, a CuPy array or a NumPy array).
"""

from __future__ import annotations

import ctypes

from . import dtypes

KDL_CPU = 1
KDL_CUDA = 2
KDL_CUDA_HOST = 3
KDL_CUDA_MANAGED = 13


class DLDevice(ctypes.Structure):
    _fields_ = [("device_type", ctypes.c_int32), ("device_id", ctypes.c_int32)]


class DLDataType(ctypes.Structure):
    _fields_ = [("code", ctypes.c_uint8), ("bits", ctypes.c_uint8), ("lanes", ctypes.c_uint16)]


class DLTensor(ctypes.Structure):
    _fields_ = [
        ("data", ctypes.c_void_p),
        ("device", DLDevice),
        ("ndim", ctypes.c_int32),
        ("dtype", DLDataType),
        ("shape", ctypes.POINTER(ctypes.c_int64)),
        ("strides", ctypes.POINTER(ctypes.c_int64)),
        ("byte_offset", ctypes.c_uint64),
    ]


class DLManagedTensor(ctypes.Structure):
    pass


_DELETER = ctypes.CFUNCTYPE(None, ctypes.POINTER(DLManagedTensor))
DLManagedTensor._fields_ = [
    ("dl_tensor", DLTensor),
    ("manager_ctx", ctypes.c_void_p),
    ("deleter", _DELETER),
]

_pyapi = ctypes.pythonapi
_pyapi.PyCapsule_GetPointer.restype = ctypes.c_void_p
_pyapi.PyCapsule_GetPointer.argtypes = [ctypes.py_object, ctypes.c_char_p]
_pyapi.PyCapsule_New.restype = ctypes.py_object
_pyapi.PyCapsule_New.argtypes = [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p]
_pyapi.PyCapsule_IsValid.restype = ctypes.c_int
_pyapi.PyCapsule_IsValid.argtypes = [ctypes.py_object, ctypes.c_char_p]


def make_dltensor(ptr: int, shape, strides, dtype: str, device_id: int, device_type: int = KDL_CUDA):
    """Builds a DLTensor (and the arrays it points to) for a raw buffer.

    Returns (tensor, keepalive): keep `keepalive` referenced while the tensor
    is in use.
    """
    nd = len(shape)
    shp = (ctypes.c_int64 * max(nd, 1))(*shape)
    std = (ctypes.c_int64 * max(nd, 1))(*strides)
    code, bits = dtypes.dl_code_bits(dtype)
    t = DLTensor()
    t.data = ctypes.c_void_p(ptr)
    t.device = DLDevice(device_type, device_id)
    t.ndim = nd
    t.dtype = DLDataType(code, bits, 1)
    t.shape = ctypes.cast(shp, ctypes.POINTER(ctypes.c_int64))
    t.strides = ctypes.cast(std, ctypes.POINTER(ctypes.c_int64))
    t.byte_offset = 0
    return t, (shp, std)


class _ForeignView:
    """A borrowed DLTensor read out of a producer's `__dlpack__` capsule."""

    __slots__ = ("capsule", "managed")

    def __init__(self, obj, stream=None):
        try:
            cap = obj.__dlpack__(stream=stream) if stream is not None else obj.__dlpack__()
        except TypeError:
            cap = obj.__dlpack__()
        if not _pyapi.PyCapsule_IsValid(cap, b"dltensor"):
            raise TypeError("object's __dlpack__ did not return a 'dltensor' capsule")
        addr = _pyapi.PyCapsule_GetPointer(cap, b"dltensor")
        self.capsule = cap  # the producer's capsule destructor frees it
        self.managed = DLManagedTensor.from_address(addr)

    @property
    def tensor(self) -> DLTensor:
        return self.managed.dl_tensor


# DLPack's C exchange API (the public struct `DLPackExchangeAPI` of DLPack 1.x,
# a capsule on the producer's type): its dltensor_from_py_object_no_sync fills a
# DLTensor in one C call, without a capsule, where __dlpack__ takes microseconds.
class _ExchangeAPI(ctypes.Structure):
    _fields_ = [
        ("major", ctypes.c_uint32),
        ("minor", ctypes.c_uint32),
        ("prev_api", ctypes.c_void_p),
        ("managed_tensor_allocator", ctypes.c_void_p),
        ("managed_tensor_from_py_object_no_sync", ctypes.c_void_p),
        ("managed_tensor_to_py_object_no_sync", ctypes.c_void_p),
        ("dltensor_from_py_object_no_sync", ctypes.c_void_p),
        ("current_work_stream", ctypes.c_void_p),
    ]


_FROM_OBJECT = ctypes.PYFUNCTYPE(ctypes.c_int, ctypes.py_object, ctypes.c_void_p)
_WORK_STREAM = ctypes.PYFUNCTYPE(ctypes.c_int, ctypes.c_int, ctypes.c_int32, ctypes.POINTER(ctypes.c_void_p))
_exchange: dict = {}  # producer type -> (from_py_object, current_work_stream) or None


def _exchange_api(cls):
    """The exchange functions of a producer type, or None (looked up once per type)."""
    if cls in _exchange:
        return _exchange[cls]
    found = None
    cap = getattr(cls, "__dlpack_c_exchange_api__", None)
    if cap is not None and _pyapi.PyCapsule_IsValid(cap, b"dlpack_exchange_api"):
        api = _ExchangeAPI.from_address(_pyapi.PyCapsule_GetPointer(cap, b"dlpack_exchange_api"))
        if api.major == 1 and api.dltensor_from_py_object_no_sync and api.current_work_stream:
            found = (_FROM_OBJECT(api.dltensor_from_py_object_no_sync), _WORK_STREAM(api.current_work_stream))
    _exchange[cls] = found
    return found


def _exchanged(obj, checked):
    """(DLTensor of `obj` through the exchange API, checked), or (None, checked)
    where it has none, fails, or has to be asked through `__dlpack__` (see
    call_tensors).  `checked`: the stream needs no look any more."""
    api = _exchange_api(type(obj))
    if api is None or getattr(obj, "requires_grad", False):
        return None, checked
    t = DLTensor()
    try:
        if api[0](obj, ctypes.addressof(t)) != 0:
            return None, checked
        if not checked:
            cur = ctypes.c_void_p()
            checked = (t.device.device_type == KDL_CUDA
                       and api[1](KDL_CUDA, t.device.device_id, ctypes.byref(cur)) == 0 and not cur.value)
    except Exception:  # what is wrong with the tensor, __dlpack__ says
        return None, checked
    return (t if checked else None), checked


def call_tensors(objs, names, stream):
    """DLTensor pointers for one call: a list of ctypes references (None for
    None) and what to keep alive until the call returns.

    Producers with the C exchange API are read through it.  That API does no
    stream synchronisation, so without an explicit `stream` (the call then runs
    on the legacy default stream) it is used only while the producer's current
    stream is that one; otherwise `__dlpack__` makes the default stream wait for
    the producer's, as it does for every other call here.  Nor does it refuse what
    `__dlpack__` does (a tensor that requires a gradient): those go that way too.
    """
    refs, keep = [], []
    checked = stream is not None
    for obj, name in zip(objs, names):
        if obj is None:
            refs.append(None)
            continue
        t, checked = _exchanged(obj, checked)
        if t is not None:
            refs.append(ctypes.byref(t))
            keep.append(t)
            continue
        ptr, k = as_dltensor(obj, name)
        refs.append(ptr)
        keep.append(k)
    return refs, keep


def as_dltensor(obj, name: str = "tensor"):
    """Returns (ctypes pointer to a DLTensor, keepalive) for `obj`."""
    from .device_array import DeviceArray, HostBuffer

    if obj is None:
        return None, None
    if isinstance(obj, DeviceArray):
        t = obj._dltensor()
        return ctypes.pointer(t), obj
    if isinstance(obj, HostBuffer):
        t, keep = obj._dltensor()
        return ctypes.pointer(t), (obj, keep)
    if hasattr(obj, "__dlpack__"):
        view = _ForeignView(obj)
        return ctypes.pointer(view.managed.dl_tensor), view
    raise TypeError(f"{name}: expected a DeviceArray or a DLPack-capable device array, got {type(obj).__name__}")


def describe(obj) -> tuple[tuple, tuple, str, int, int]:
    """(shape, strides in elements, dtype name, device_type, device_id) of any accepted array."""
    ptr, keep = as_dltensor(obj)
    t = ptr.contents
    nd = t.ndim
    shape = tuple(t.shape[i] for i in range(nd))
    if t.strides:
        strides = tuple(t.strides[i] for i in range(nd))
    else:
        acc, st = 1, []
        for s in reversed(shape):
            st.append(acc)
            acc *= s
        strides = tuple(reversed(st))
    dt = dtypes.from_dl(t.dtype.code, t.dtype.bits)
    del keep
    return shape, strides, dt, t.device.device_type, t.device.device_id

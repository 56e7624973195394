"""ctypes binding of libflagcx_amd.so (include/flagcx_amd.h).

Device memory and streams come from torch; nothing here computes.  Every call
goes through the C ABI, and a missing library is an error (ImportError-like
RuntimeError), never a silent fallback.
"""
import ctypes as C
import enum
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(HERE, "lib", "libflagcx_amd.so")
_lib = None

MAX_RANKS = 64
CHUNKSIZE = 4 * 1024 * 1024


class Result(enum.IntEnum):          # flagcx/include/flagcx.h:12-24
    Success = 0
    UnhandledDeviceError = 1
    SystemError = 2
    InternalError = 3
    InvalidArgument = 4
    InvalidUsage = 5
    RemoteError = 6
    InProgress = 7
    UnhandledCCLError = 8
    NotSupported = 9


class DataType(enum.IntEnum):        # flagcx/include/flagcx.h:27-44
    Int8 = 0
    Uint8 = 1
    Int32 = 2
    Uint32 = 3
    Int64 = 4
    Uint64 = 5
    Float16 = 6
    Float32 = 7
    Float64 = 8
    Bfloat16 = 9


class RedOp(enum.IntEnum):           # flagcx/include/flagcx.h:47-57
    Sum = 0
    Prod = 1
    Max = 2
    Min = 3
    Avg = 4


class FlagcxError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__("flagcx result %d (%s): %s" % (code, Result(code).name if 0 <= code < 10 else "?", msg))
        self.code = code


class Stream(C.Structure):
    """struct flagcxStream { hipStream_t base; } (flagcx/adaptor/include/amd_adaptor.h:14-16)"""
    _fields_ = [("base", C.c_void_p)]


class ReduceArgs(C.Structure):       # flagcxLocalReduceArgs
    _fields_ = [("sendbuffs", C.POINTER(C.c_void_p)), ("recvbuff", C.c_void_p), ("count", C.c_uint64),
                ("nranks", C.c_int32), ("datatype", C.c_int32), ("op", C.c_int32), ("result", C.c_int32)]


class ReduceDesc(C.Structure):       # flagcxLocalReduceDesc
    _fields_ = [("sendbuffs", C.POINTER(C.c_void_p)), ("recvbuff", C.c_void_p), ("count", C.c_size_t)]


class FanoutDesc(C.Structure):       # flagcxLocalFanoutDesc
    _fields_ = [("src", C.c_void_p), ("dsts", C.POINTER(C.c_void_p)), ("ndsts", C.c_int), ("bytes", C.c_size_t)]


NORM_POST = 1                        # FLAGCX_LOCAL_NORM_POST
NORM_PRE = 2                         # FLAGCX_LOCAL_NORM_PRE
NORM_MAX_DIM = 16384


class BlockEnd(C.Structure):         # flagcxLocalBlockEnd
    _fields_ = [("rows", C.c_size_t), ("dim", C.c_size_t), ("norms", C.c_int), ("datatype", C.c_int),
                ("residualtype", C.c_int), ("weighttype", C.c_int), ("scale", C.c_float), ("eps", C.c_float),
                ("weightoffset", C.c_float), ("postweight", C.c_void_p), ("preweight", C.c_void_p), ("gate", C.c_void_p),
                ("gatestride", C.c_size_t), ("gaterows", C.c_size_t)]


class ReduceTrigger(C.Structure):    # flagcxLocalReduceTrigger, 16-byte aligned
    _fields_ = [("value", C.c_uint64 * 4)]
    _pack_ = 16

    @classmethod
    def make(cls, addr1, addr2, addr3, count, datatype, redop, nthreads=0):
        t = cls()
        t.value[0], t.value[1], t.value[2] = addr1, addr2, addr3
        t.value[3] = (count & 0xffffffff) | ((nthreads & 0xffff) << 32) | ((int(datatype) & 0xf) << 48) | \
                     ((int(redop) & 0xf) << 52)
        return t


class DeviceTrigger(C.Structure):    # flagcxLocalDeviceTrigger
    _fields_ = [("fst", C.c_uint64), ("snd", C.c_uint64)]

    @property
    def addr(self):
        return self.fst

    @property
    def count(self):
        return self.snd & 0xffffffff

    @property
    def peer(self):
        return (self.snd >> 32) & 0xfffff

    @property
    def datatype(self):
        return (self.snd >> 52) & 0xf

    @property
    def prim(self):
        return (self.snd >> 56) & 0xf


class CopyArgs(C.Structure):         # flagcxLocalCopyArgs
    _fields_ = [("dst", C.c_void_p), ("src", C.c_void_p), ("size", C.c_uint64), ("result", C.c_int32),
                ("reserved", C.c_int32)]


EXPORTS = [
    "flagcxLocalGetDataTypeSize", "flagcxLocalInit", "flagcxLocalGetErrorString", "flagcxLocalGetLastError",
    "flagcxLocalTune", "flagcxLocalGetTune", "flagcxLocalTuneLoads", "flagcxLocalGetTuneLoads", "flagcxLocalPlaceBuffers", "flagcxLocalReduce", "flagcxLocalReduceScatter", "flagcxLocalReduceScatterChunked",
    "flagcxLocalAllReduce", "flagcxLocalRingChunkTable", "flagcxLocalMemcpy", "flagcxLocalMemset",
    "flagcxLocalRefresh", "flagcxLocalPack", "flagcxLocalUnpack", "flagcxLocalPackList",
    "flagcxLocalUnpackList", "flagcxLocalCopyFanout", "flagcxLocalReduceFunc", "flagcxLocalCopyFunc",
    "flagcxLocalSetMaxSpinCount", "deviceAsyncStore", "deviceAsyncLoad",
    "flagcxLocalReduceBatch", "flagcxLocalReduceBatchSparse", "flagcxLocalReduceTriggers",
    "flagcxLocalGateCreate", "flagcxLocalGateDestroy", "flagcxLocalReduceBatchGated", "flagcxLocalGateOpen",
    "flagcxLocalGateQuery", "flagcxLocalGateOwnStream",
    "flagcxLocalFifoInit", "flagcxLocalFifoDestroy", "flagcxLocalFifoDequeue", "flagcxLocalP2pDemo",
    "flagcxLocalRingCreate", "flagcxLocalRingDestroy", "flagcxLocalRingSendRecv",
    "flagcxLocalRingReduceScatter",
    "flagcxLocalGetDeviceAdaptor", "flagcxLocalDeviceAdaptorLayout",
    "flagcxLocalPlanCreate", "flagcxLocalPlanDestroy", "flagcxLocalPlanImportXml", "flagcxLocalPlanExportXml",
    "flagcxLocalPlanSetAlgorithm", "flagcxLocalPlanSetFused", "flagcxLocalPlanGetTraffic", "flagcxLocalPlanSetChunks", "flagcxLocalPlanSetAlltoAllv", "flagcxLocalPlanExecute", "flagcxLocalPlanGetLastError",
    "flagcxLocalReduceFifoCreate", "flagcxLocalReduceFifoDestroy", "flagcxLocalReduceFifoStart",
    "flagcxLocalReduceFifoStop", "flagcxLocalReduceFifoEnqueue", "flagcxLocalReduceFifoEnqueueReduce",
    "flagcxLocalReduceFifoQuery", "flagcxLocalReduceFifoWait", "flagcxLocalReduceFifoGetGrid",
    "flagcxLocalReduceFifoSetWaves", "flagcxLocalReduceFifoSetLinger", "flagcxLocalReduceFifoSetOwnQueue", "flagcxLocalReduceFifoSetWindow", "flagcxLocalReduceFifoGetType", "flagcxLocalRingReduceScatterFifo",
    "flagcxLocalReduceFifoGetLastError", "flagcxLocalStagedReduceScatterNoAlloc",
    "flagcxLocalReduceNorm", "flagcxLocalReduceNormBackward", "flagcxLocalReduceNormBackwardWorkspace",
    "flagcxLocalEmbedding", "flagcxLocalEmbeddingGrad", "flagcxLocalEmbeddingGradWorkspace",
]


def lib_path():
    return _LIB_PATH


def lib():
    """The loaded C library; raises if it was not built (python -m flagcx_amd.build)."""
    global _lib
    if _lib is None:
        if not os.path.exists(_LIB_PATH):
            raise RuntimeError("%s is missing: build it with `python -m flagcx_amd.build` "
                               "(there is no fallback implementation)" % _LIB_PATH)
        # PyTorch ships its own copy of the HIP runtime.  Whichever copy a process loads first serves both,
        # and PyTorch does not find its GPUs through another one: where torch is in the process, let it
        # load and initialise its runtime before this library brings in the system's (torch may be imported
        # later by the same process: tests, bench.py and every user of this binding hold their buffers in it).
        try:
            import torch
            torch.cuda.is_available()
        except Exception:
            pass
        L = C.CDLL(_LIB_PATH)
        vp, sz, i, pp = C.c_void_p, C.c_size_t, C.c_int, C.POINTER(C.c_void_p)
        sp = C.POINTER(Stream)
        L.flagcxLocalGetDataTypeSize.restype = sz
        L.flagcxLocalGetDataTypeSize.argtypes = [i]
        L.flagcxLocalInit.argtypes = []
        L.flagcxLocalGetErrorString.restype = C.c_char_p
        L.flagcxLocalGetErrorString.argtypes = [i]
        L.flagcxLocalGetLastError.restype = C.c_char_p
        L.flagcxLocalTune.argtypes = [i, i]
        L.flagcxLocalPlaceBuffers.argtypes = [vp, sz, sz, i, pp]
        L.flagcxLocalGetTune.argtypes = [i, C.POINTER(i)]
        L.flagcxLocalTuneLoads.argtypes = [i, i]
        L.flagcxLocalGetTuneLoads.argtypes = [i, C.POINTER(i)]
        L.flagcxLocalReduce.argtypes = [pp, i, vp, sz, i, i, sp]
        L.flagcxLocalReduceScatter.argtypes = [pp, i, i, vp, sz, i, i, sp]
        L.flagcxLocalReduceScatterChunked.argtypes = [pp, i, i, vp, sz, i, i, sz, sp]
        L.flagcxLocalAllReduce.argtypes = [pp, i, vp, sz, i, i, sp]
        L.flagcxLocalRingChunkTable.argtypes = [sz, i, i, C.POINTER(sz), C.POINTER(sz)]
        L.flagcxLocalMemcpy.argtypes = [vp, vp, sz, sp]
        L.flagcxLocalMemset.argtypes = [vp, i, sz, sp]
        L.flagcxLocalRefresh.argtypes = [vp, sz, sz, sz, sz, i, i, sp]
        L.flagcxLocalPack.argtypes = [vp, vp, sz, sz, sz, sp]
        L.flagcxLocalUnpack.argtypes = [vp, vp, sz, sz, sz, sp]
        L.flagcxLocalPackList.argtypes = [vp, pp, i, sz, sp]
        L.flagcxLocalUnpackList.argtypes = [pp, vp, i, sz, sp]
        L.flagcxLocalCopyFanout.argtypes = [C.POINTER(FanoutDesc), i, sp]
        ep, i64, f = C.POINTER(BlockEnd), C.c_int64, C.c_float
        L.flagcxLocalReduceNorm.argtypes = [ep, pp, i, sz, vp, sz, vp, sz, vp, sz, vp, sz, sp]
        L.flagcxLocalReduceNormBackward.argtypes = [ep, vp, sz, vp, sz, vp, sz, vp, sz, vp, sz, vp, sz, vp, vp, vp, sz,
                                                    vp, sz, sp]
        L.flagcxLocalReduceNormBackwardWorkspace.argtypes = [ep, C.POINTER(sz)]
        L.flagcxLocalEmbedding.argtypes = [vp, i, sz, sz, sz, vp, i, sz, i64, f, vp, i, sz, sp]
        L.flagcxLocalEmbeddingGrad.argtypes = [vp, i, sz, vp, i, sz, i64, f, vp, i, sz, sz, sz, i, vp, sz, sp]
        L.flagcxLocalEmbeddingGradWorkspace.argtypes = [sz, sz, sz, C.POINTER(sz)]
        L.flagcxLocalReduceFunc.restype = None
        L.flagcxLocalReduceFunc.argtypes = [sp, C.POINTER(ReduceArgs)]
        L.flagcxLocalCopyFunc.restype = None
        L.flagcxLocalCopyFunc.argtypes = [sp, C.POINTER(CopyArgs)]
        L.flagcxLocalReduceBatch.argtypes = [C.POINTER(ReduceDesc), i, i, i, i, sp]
        L.flagcxLocalReduceBatchSparse.argtypes = [C.POINTER(ReduceDesc), i, i, i, i, i, sp]
        L.flagcxLocalReduceTriggers.argtypes = [C.POINTER(ReduceTrigger), i, sp]
        L.flagcxLocalFifoInit.argtypes = [C.POINTER(vp)]
        L.flagcxLocalFifoDestroy.argtypes = [vp]
        L.flagcxLocalFifoDequeue.argtypes = [vp, C.POINTER(DeviceTrigger)]
        L.flagcxLocalP2pDemo.argtypes = [vp, vp, sz, i, i, i, vp, sp]
        L.flagcxLocalRingCreate.argtypes = [C.POINTER(vp), vp, sz, i, sz, i]
        L.flagcxLocalRingDestroy.argtypes = [vp]
        L.flagcxLocalRingSendRecv.argtypes = [vp, vp, vp, sz, sp, sp]
        L.flagcxLocalRingReduceScatter.argtypes = [vp, pp, i, i, vp, sz, i, i, sp, sp]
        L.flagcxLocalStagedReduceScatterNoAlloc.argtypes = [pp, i, i, vp, sz, i, i, sp]
        L.flagcxLocalGetDeviceAdaptor.restype = vp
        L.flagcxLocalGetDeviceAdaptor.argtypes = []
        L.flagcxLocalDeviceAdaptorLayout.argtypes = [C.POINTER(sz), i]
        L.flagcxLocalPlanCreate.argtypes = [C.POINTER(vp), i, C.POINTER(i), C.POINTER(i), sz, i, i]
        L.flagcxLocalPlanDestroy.argtypes = [vp]
        L.flagcxLocalPlanImportXml.argtypes = [vp, C.c_char_p]
        L.flagcxLocalPlanExportXml.argtypes = [vp, C.c_char_p]
        L.flagcxLocalPlanSetAlgorithm.argtypes = [vp, i]
        L.flagcxLocalPlanSetFused.argtypes = [vp, i]
        L.flagcxLocalPlanGetTraffic.argtypes = [vp, C.POINTER(C.c_uint64), C.POINTER(C.c_uint64)]
        L.flagcxLocalPlanSetChunks.argtypes = [vp, sz]
        szp = C.POINTER(C.c_size_t)
        L.flagcxLocalPlanSetAlltoAllv.argtypes = [vp, szp, szp, szp, szp]
        L.flagcxLocalPlanExecute.argtypes = [vp, pp, pp, pp, i, i, sp]
        L.flagcxLocalPlanGetLastError.restype = C.c_char_p
        L.flagcxLocalPlanGetLastError.argtypes = [vp]
        u64p = C.POINTER(C.c_uint64)
        L.flagcxLocalReduceFifoCreate.argtypes = [C.POINTER(vp), i, i, i, i]
        L.flagcxLocalReduceFifoDestroy.argtypes = [vp]
        L.flagcxLocalReduceFifoStart.argtypes = [vp]
        L.flagcxLocalReduceFifoStop.argtypes = [vp]
        L.flagcxLocalReduceFifoEnqueue.argtypes = [vp, C.POINTER(ReduceTrigger), u64p]
        L.flagcxLocalReduceFifoEnqueueReduce.argtypes = [vp, pp, i, vp, sz, u64p]
        L.flagcxLocalReduceFifoQuery.argtypes = [vp, u64p, u64p, C.POINTER(i)]
        L.flagcxLocalReduceFifoSetOwnQueue.argtypes = [vp, i]
        L.flagcxLocalGateCreate.argtypes = [pp]
        L.flagcxLocalGateDestroy.argtypes = [vp]
        L.flagcxLocalReduceBatchGated.argtypes = [vp, C.POINTER(ReduceDesc), i, i, i, i, sp, u64p]
        L.flagcxLocalGateOpen.argtypes = [vp, C.c_uint64]
        L.flagcxLocalGateQuery.argtypes = [vp, u64p, u64p, C.POINTER(i)]
        L.flagcxLocalGateOwnStream.argtypes = [vp, C.POINTER(sp)]
        L.flagcxLocalReduceFifoWait.argtypes = [vp, C.c_uint64]
        L.flagcxLocalReduceFifoGetGrid.argtypes = [vp, C.POINTER(C.c_uint)]
        L.flagcxLocalReduceFifoSetWaves.argtypes = [vp, i]
        L.flagcxLocalReduceFifoSetLinger.argtypes = [vp, C.c_int64]
        L.flagcxLocalReduceFifoSetWindow.argtypes = [vp, sz]
        L.flagcxLocalReduceFifoGetType.argtypes = [vp, C.POINTER(i), C.POINTER(i), C.POINTER(i)]
        L.flagcxLocalRingReduceScatterFifo.argtypes = [vp, vp, pp, i, i, vp, sz, sp]
        L.flagcxLocalReduceFifoGetLastError.restype = C.c_char_p
        L.flagcxLocalReduceFifoGetLastError.argtypes = [vp]
        L.flagcxLocalSetMaxSpinCount.restype = None
        L.flagcxLocalSetMaxSpinCount.argtypes = [C.c_int64]
        for name in ("deviceAsyncStore", "deviceAsyncLoad"):
            fn = getattr(L, name)
            fn.restype = None
            fn.argtypes = [sp, vp]
        _lib = L
    return _lib


def check(code):
    if code != 0:
        raise FlagcxError(code, lib().flagcxLocalGetLastError().decode())


def type_size(dtype):
    return lib().flagcxLocalGetDataTypeSize(int(dtype))


# ---------------------------------------------------------------- torch side

def _torch():
    import torch
    return torch


def dtype_of(t, bits_as=None):
    """flagcx enum for a torch tensor's dtype (uint16/uint32/uint64 carried as the
    signed tensor type of the same width unless bits_as names the enum)."""
    torch = _torch()
    if bits_as is not None:
        return DataType(bits_as)
    m = {torch.int8: DataType.Int8, torch.uint8: DataType.Uint8, torch.int32: DataType.Int32,
         torch.int64: DataType.Int64, torch.float16: DataType.Float16, torch.float32: DataType.Float32,
         torch.float64: DataType.Float64, torch.bfloat16: DataType.Bfloat16}
    return m[t.dtype]


def current_stream():
    """A flagcxStream wrapper around torch's current HIP stream (not owned)."""
    torch = _torch()
    return Stream(torch.cuda.current_stream().cuda_stream)


def _sref(stream):
    return C.byref(stream) if stream is not None else None


def _ptr_array(ptrs):
    return (C.c_void_p * len(ptrs))(*ptrs)


def place_buffers(pool_ptr, pool_bytes, nbytes, n):
    """Addresses for n buffers of nbytes inside the pool, in different HBM channel groups."""
    out = (C.c_void_p * n)()
    check(lib().flagcxLocalPlaceBuffers(pool_ptr, pool_bytes, nbytes, n, out))
    return [int(p) for p in out]


def reduce(srcs, dst, op, dtype=None, count=None, stream="current"):
    """dst = fold of srcs (torch device tensors) through flagcxLocalReduce."""
    st = current_stream() if stream == "current" else stream
    dt = dtype_of(dst, dtype)
    n = dst.numel() if count is None else count
    check(lib().flagcxLocalReduce(_ptr_array([s.data_ptr() for s in srcs]), len(srcs), dst.data_ptr(), n,
                                  int(dt), int(op), _sref(st)))
    return dst


def reduce_scatter(sendbuffs, rank, recv, op, dtype=None, chunkbytes=None, stream="current"):
    st = current_stream() if stream == "current" else stream
    dt = dtype_of(recv, dtype)
    ptrs = _ptr_array([s.data_ptr() for s in sendbuffs])
    if chunkbytes is None:
        check(lib().flagcxLocalReduceScatter(ptrs, len(sendbuffs), rank, recv.data_ptr(), recv.numel(),
                                             int(dt), int(op), _sref(st)))
    else:
        check(lib().flagcxLocalReduceScatterChunked(ptrs, len(sendbuffs), rank, recv.data_ptr(), recv.numel(),
                                                    int(dt), int(op), chunkbytes, _sref(st)))
    return recv


STATIC_STAGING_BYTES = 8 * 1024 * 1024


def staged_reduce_scatter_noalloc(sendbuffs, rank, recv, op, dtype=None, stream="current"):
    """flagcxLocalStagedReduceScatterNoAlloc: peers' slices staged in the library's static area."""
    st = current_stream() if stream == "current" else stream
    dt = dtype_of(recv, dtype)
    check(lib().flagcxLocalStagedReduceScatterNoAlloc(_ptr_array([s.data_ptr() for s in sendbuffs]), len(sendbuffs),
                                                      rank, recv.data_ptr(), recv.numel(), int(dt), int(op),
                                                      _sref(st)))
    return recv


def all_reduce(sendbuffs, recv, op, dtype=None, stream="current"):
    st = current_stream() if stream == "current" else stream
    dt = dtype_of(recv, dtype)
    check(lib().flagcxLocalAllReduce(_ptr_array([s.data_ptr() for s in sendbuffs]), len(sendbuffs),
                                     recv.data_ptr(), recv.numel(), int(dt), int(op), _sref(st)))
    return recv


def reduce_batch(descs, op, dtype, nranks, stream="current"):
    """descs: list of (list_of_src_ptrs, dst_ptr, count).  One flagcxLocalReduceBatch call."""
    st = current_stream() if stream == "current" else stream
    keep = [_ptr_array(list(d[0])) for d in descs]
    arr = (ReduceDesc * len(descs))(*[ReduceDesc(keep[i], d[1], d[2]) for i, d in enumerate(descs)])
    check(lib().flagcxLocalReduceBatch(arr, len(descs), nranks, int(dtype), int(op), _sref(st)))


def reduce_batch_sparse(descs, op, dtype, nlive, nzero, stream="current"):
    """descs as reduce_batch, each listing the nlive members that hold data; nzero more members hold zeros."""
    st = current_stream() if stream == "current" else stream
    keep = [_ptr_array(list(d[0])) for d in descs]
    arr = (ReduceDesc * len(descs))(*[ReduceDesc(keep[i], d[1], d[2]) for i, d in enumerate(descs)])
    check(lib().flagcxLocalReduceBatchSparse(arr, len(descs), nlive, nzero, int(dtype), int(op), _sref(st)))


def reduce_triggers(triggers, stream="current"):
    st = current_stream() if stream == "current" else stream
    arr = (ReduceTrigger * len(triggers))(*triggers)
    check(lib().flagcxLocalReduceTriggers(arr, len(triggers), _sref(st)))


def ring_chunk_table(count, dtype, nranks):
    off = (C.c_size_t * nranks)()
    ln = (C.c_size_t * nranks)()
    check(lib().flagcxLocalRingChunkTable(count, int(dtype), nranks, off, ln))
    return list(off), list(ln)


def memcpy(dst_ptr, src_ptr, size, stream="current"):
    st = current_stream() if stream == "current" else stream
    check(lib().flagcxLocalMemcpy(dst_ptr, src_ptr, size, _sref(st)))


def memset(ptr, value, size, stream="current"):
    st = current_stream() if stream == "current" else stream
    check(lib().flagcxLocalMemset(ptr, value, size, _sref(st)))


def refresh(buff, start, offset, count, totalcount, op, dtype=None, stream="current"):
    st = current_stream() if stream == "current" else stream
    dt = dtype_of(buff, dtype)
    check(lib().flagcxLocalRefresh(buff.data_ptr(), start, offset, count, totalcount, int(dt), int(op), _sref(st)))


def pack(dst_ptr, src_ptr, nchunks, chunkbytes, srcstride, stream="current"):
    st = current_stream() if stream == "current" else stream
    check(lib().flagcxLocalPack(dst_ptr, src_ptr, nchunks, chunkbytes, srcstride, _sref(st)))


def unpack(dst_ptr, src_ptr, nchunks, chunkbytes, dststride, stream="current"):
    st = current_stream() if stream == "current" else stream
    check(lib().flagcxLocalUnpack(dst_ptr, src_ptr, nchunks, chunkbytes, dststride, _sref(st)))


def pack_list(dst_ptr, src_ptrs, nbytes, stream="current"):
    st = current_stream() if stream == "current" else stream
    check(lib().flagcxLocalPackList(dst_ptr, _ptr_array(src_ptrs), len(src_ptrs), nbytes, _sref(st)))


def unpack_list(dst_ptrs, src_ptr, nbytes, stream="current"):
    st = current_stream() if stream == "current" else stream
    check(lib().flagcxLocalUnpackList(_ptr_array(dst_ptrs), src_ptr, len(dst_ptrs), nbytes, _sref(st)))


def copy_fanout(copies, stream="current"):
    """copies: list of (src_ptr, list_of_dst_ptrs, nbytes).  One flagcxLocalCopyFanout call."""
    st = current_stream() if stream == "current" else stream
    keep = [_ptr_array(list(c[1])) for c in copies]
    arr = (FanoutDesc * len(copies))(*[FanoutDesc(c[0], keep[i], len(c[1]), c[2]) for i, c in enumerate(copies)])
    check(lib().flagcxLocalCopyFanout(arr, len(copies), _sref(st)))


# ------------------------------------------- the residual stream of a tensor-parallel model
# Matrices are 2-d tensors with rows of consecutive elements (a row stride of their own is
# fine) on the current device.  Outputs are given by the caller and returned.

def _refuse(msg):
    raise FlagcxError(int(Result.InvalidArgument), msg)


def _size(name, n):
    """n, which ctypes would cut to 64 bits without a word."""
    if not 0 <= n < 1 << 64:
        _refuse("%s %d" % (name, n))
    return n


def _rows(name, t, shape, dtype, device):
    """(address, row stride in elements) of a matrix; (None, 0) for None.  device is an index."""
    if t is None:
        return None, 0
    if t.shape == shape and t.dtype is dtype and t.get_device() == device and t.is_contiguous():
        return t.data_ptr(), 0
    if t.dtype is not dtype or t.get_device() != device:
        _refuse("%s: %s on %s, expected %s on cuda:%d" % (name, t.dtype, t.device, dtype, device))
    if t.shape != shape:
        _refuse("%s: shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))
    s0, s1 = t.stride()
    rows, dim = shape
    if s1 != 1 and dim > 1:
        _refuse("%s: elements of a row are not consecutive" % name)
    if rows <= 1:
        return t.data_ptr(), 0
    if s0 < dim:
        _refuse("%s: row stride %d below %d" % (name, s0, dim))
    return t.data_ptr(), s0


def _vector(name, t, n, dtype, device):
    if t is None:
        return None
    if t.dtype is not dtype or t.get_device() != device:
        _refuse("%s: %s on %s, expected %s on cuda:%d" % (name, t.dtype, t.device, dtype, device))
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        _refuse("%s: expected %d consecutive elements" % (name, n))
    return t.data_ptr()


def _gates(name, t, rows, dim, gate_rows, dtype, device):
    """Like _rows, for one row of gates for all rows (a vector will do) or one for every gate_rows of them."""
    if t is None:
        return None, 0
    if _size("gate_rows", gate_rows) == 0 and t.dim() == 1:
        return _vector(name, t, dim, dtype, device), 0
    return _rows(name, t, (-(-rows // gate_rows) if gate_rows else 1, dim), dtype, device)


def _device(t):
    """Index of a call's device: that of t, which has to be the current one."""
    d = t.get_device()
    if d < 0 or d != _torch()._C._cuda_getDevice():
        _refuse("tensors on %s, which is not the current device" % t.device)
    return d


def _stream_ref(stream, device):
    """The stream argument of a call on `device`, by reference."""
    if stream == "current":
        return C.byref(Stream(_torch()._C._cuda_getCurrentRawStream(device)))
    return _sref(stream)


def _workspace(ws, need, device, stream):
    """(address, bytes, owner) of the workspace; allocated on the current stream where none is given."""
    if ws is None:
        if need == 0:
            return None, 0, None
        if stream != "current":
            _refuse("a call on a stream of its own needs its own workspace")
        torch = _torch()
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        return ws.data_ptr(), need, ws
    if ws.get_device() != device or not ws.is_contiguous():
        _refuse("workspace: not a contiguous tensor on cuda:%d" % device)
    return ws.data_ptr(), ws.numel() * ws.element_size(), ws


def _block_end(rows, dim, act, res, device, post_weight, pre_weight, gate, gate_rows, scale, eps, weight_offset,
               post, pre):
    w = post_weight if post_weight is not None else pre_weight
    wt = w.dtype if w is not None else act
    types = _float_types()
    if act not in types or res not in types or wt not in types:
        _refuse("data types %s, %s, %s" % (act, res, wt))
    gp, gs = _gates("gate", gate, rows, dim, gate_rows, act, device)
    return BlockEnd(rows, dim, (NORM_POST if post else 0) | (NORM_PRE if pre else 0), types[act], types[res], types[wt],
                    scale, eps, weight_offset, _vector("post_weight", post_weight, dim, wt, device),
                    _vector("pre_weight", pre_weight, dim, wt, device), gp, gs, gate_rows if gate is not None else 0)


_FLOAT_TYPES = {}


def _float_types():
    if not _FLOAT_TYPES:
        torch = _torch()
        _FLOAT_TYPES.update({torch.float16: 6, torch.float32: 7, torch.bfloat16: 9})
    return _FLOAT_TYPES


def reduce_norm(srcs, residual, residual_out, norm_out=None, sum_out=None, post_weight=None, pre_weight=None, gate=None,
                gate_rows=0, scale=1.0, eps=1e-6, weight_offset=0.0, post_norm=None, stream="current"):
    """flagcxLocalReduceNorm: the end of a tensor-parallel block.

    s = sum of srcs (-> sum_out); u = s, or its RMS norm where post_norm says so (default: where there is a
    post_weight); residual_out = residual + scale * gate * u; norm_out = RMS norm of that, if given.
    gate: (dim,) or (1, dim) for all rows, or with gate_rows = n one row of gates for every n rows.  A weight
    whose norm is not there (post_weight with post_norm=False, pre_weight without a norm_out) is not read.
    Returns (residual_out, norm_out, sum_out)."""
    if not srcs:
        _refuse("no srcs")
    device = _device(residual_out)
    shape = residual_out.shape
    if len(shape) != 2:
        _refuse("residual_out: expected a matrix")
    rows, dim = shape
    act, res = srcs[0].dtype, residual_out.dtype
    ptrs, stride = [], None
    for t in srcs:
        p, st = _rows("a source", t, shape, act, device)
        if st != stride and stride is not None and (st or dim) != (stride or dim):
            _refuse("sources of different row strides")
        ptrs.append(p)
        stride = st
    end = _block_end(rows, dim, act, res, device, post_weight, pre_weight, gate, gate_rows, scale, eps, weight_offset,
                     post_weight is not None if post_norm is None else post_norm, norm_out is not None)
    rp, rs = _rows("residual", residual, shape, res, device)
    op, os_ = _rows("residual_out", residual_out, shape, res, device)
    yp, ys = _rows("norm_out", norm_out, shape, act, device)
    sp, ss = _rows("sum_out", sum_out, shape, act, device)
    check(lib().flagcxLocalReduceNorm(end, _ptr_array(ptrs), len(ptrs), stride, rp, rs, op, os_, yp, ys, sp, ss,
                                      _stream_ref(stream, device)))
    return residual_out, norm_out, sum_out


def reduce_norm_backward(residual_out, norm_grad, residual_out_grad, send_grad=None, residual_grad=None, total=None,
                         post_weight=None, pre_weight=None, gate=None, gate_rows=0, post_weight_grad=None,
                         pre_weight_grad=None, gate_grad=None, scale=1.0, eps=1e-6, weight_offset=0.0, post_norm=None,
                         dtype=None, workspace=None, stream="current"):
    """flagcxLocalReduceNormBackward.  residual_out and total are the forward pass's residual_out and sum_out,
    norm_grad and residual_out_grad the gradients of its outputs (None: zeros; with neither a norm_grad nor a
    pre_weight_grad the norm before the next block takes no part).  send_grad (the gradient of every source), residual_grad,
    post_weight_grad, pre_weight_grad and gate_grad are written where given.  dtype: the activations' type,
    where no tensor says it.  workspace: see reduce_norm_backward_workspace."""
    lead = residual_out if residual_out is not None else residual_out_grad
    if lead is None:
        lead = norm_grad
    if lead is None or lead.dim() != 2:
        _refuse("no matrix to begin from")
    device = _device(lead)
    shape = lead.shape
    rows, dim = shape
    for t in (norm_grad, total, send_grad, gate):
        if t is not None and dtype is None:
            dtype = t.dtype
    act = dtype if dtype is not None else lead.dtype
    res = residual_out_grad.dtype if residual_out_grad is not None else \
        residual_out.dtype if residual_out is not None else act
    pre = norm_grad is not None or pre_weight_grad is not None  # whether the norm before the next block has a part in it
    if not pre:
        pre_weight = None
    end = _block_end(rows, dim, act, res, device, post_weight, pre_weight, gate, gate_rows, scale, eps, weight_offset,
                     post_weight is not None if post_norm is None else post_norm, pre)
    wt = post_weight.dtype if post_weight is not None else pre_weight.dtype if pre_weight is not None else act
    tp, ts = _rows("total", total, shape, act, device)
    hp, hs = _rows("residual_out", residual_out, shape, res, device)
    yp, ys = _rows("norm_grad", norm_grad, shape, act, device)
    gp, gs = _rows("residual_out_grad", residual_out_grad, shape, res, device)
    dp, ds = _rows("send_grad", send_grad, shape, act, device)
    rp, rs = _rows("residual_grad", residual_grad, shape, res, device)
    w1 = _vector("post_weight_grad", post_weight_grad, dim, wt, device)
    w2 = _vector("pre_weight_grad", pre_weight_grad, dim, wt, device)
    ap, as_ = _gates("gate_grad", gate_grad, rows, dim, gate_rows, act, device)
    need = C.c_size_t()
    check(lib().flagcxLocalReduceNormBackwardWorkspace(end, C.byref(need)))
    wp, wb, keep = _workspace(workspace, need.value, device, stream)
    check(lib().flagcxLocalReduceNormBackward(end, tp, ts, hp, hs, yp, ys, gp, gs, dp, ds, rp, rs, w1, w2, ap, as_, wp, wb,
                                              _stream_ref(stream, device)))
    return send_grad, residual_grad


def reduce_norm_backward_workspace(rows, dim, gate=False, gate_rows=0):
    """Bytes of workspace of reduce_norm_backward; those of the longest batch do for every shorter one."""
    end = BlockEnd(_size("rows", rows), _size("dim", dim), NORM_POST | NORM_PRE, 7, 7, 7, 1.0, 1.0, 0.0, None, None,
                   1 if gate else None, 0, _size("gate_rows", gate_rows))
    need = C.c_size_t()
    check(lib().flagcxLocalReduceNormBackwardWorkspace(end, C.byref(need)))
    return need.value


def _ids(ids, device):
    torch = _torch()
    wide = ids.dtype is torch.int64
    if not wide and ids.dtype is not torch.int32 or ids.get_device() != device or not ids.is_contiguous():
        _refuse("ids: expected consecutive int32 or int64 values on cuda:%d" % device)
    return ids.data_ptr(), 4 if wide else 2, ids.numel()


def _first(first):
    if not -1 << 63 <= first < 1 << 63:
        _refuse("first: %d is no 64-bit id" % first)
    return first


def embedding(table, ids, out, first=0, scale=1.0, stream="current"):
    """flagcxLocalEmbedding: out[t] = scale * table[ids[t] - first], zeros where the table (one rank's shard of
    the vocabulary, from id `first` on) has no such row (nor any, for a padding id such as -1).  Returns out."""
    types = _float_types()
    device = _device(out)
    tt, ot, shape = table.dtype, out.dtype, table.shape
    if len(shape) != 2 or tt not in types or ot not in types:
        _refuse("table: expected a matrix of fp16, bf16 or fp32, like out")
    ip, it, tokens = _ids(ids, device)
    vocab, dim = shape
    tp, ts = _rows("table", table, shape, tt, device)
    op, os_ = _rows("out", out, (tokens, dim), ot, device)
    check(lib().flagcxLocalEmbedding(tp, types[tt], vocab, dim, ts, ip, it, tokens, _first(first), scale, op, types[ot], os_,
                                     _stream_ref(stream, device)))
    return out


def embedding_grad(out_grad, ids, table_grad, first=0, scale=1.0, accumulate=False, workspace=None, stream="current"):
    """flagcxLocalEmbeddingGrad: the gradient of embedding()'s table, written over table_grad or added to it.
    workspace: see embedding_grad_workspace.  Returns table_grad."""
    types = _float_types()
    device = _device(table_grad)
    tt, ot, shape = table_grad.dtype, out_grad.dtype, table_grad.shape
    if len(shape) != 2 or tt not in types or ot not in types:
        _refuse("table_grad: expected a matrix of fp16, bf16 or fp32, like out_grad")
    ip, it, tokens = _ids(ids, device)
    vocab, dim = shape
    tp, ts = _rows("table_grad", table_grad, shape, tt, device)
    gp, gs = _rows("out_grad", out_grad, (tokens, dim), ot, device)
    wp, wb, keep = _workspace(workspace, embedding_grad_workspace(tokens, vocab, dim), device, stream)
    check(lib().flagcxLocalEmbeddingGrad(gp, types[ot], gs, ip, it, tokens, _first(first), scale, tp, types[tt], vocab, dim,
                                         ts, 1 if accumulate else 0, wp, wb, _stream_ref(stream, device)))
    return table_grad


def embedding_grad_workspace(tokens, vocab, dim):
    """Bytes of workspace of embedding_grad; those of the largest call do for every smaller one."""
    need = C.c_size_t()
    check(lib().flagcxLocalEmbeddingGradWorkspace(_size("tokens", tokens), _size("vocab", vocab), _size("dim", dim),
                                                  C.byref(need)))
    return need.value


class Plan:
    """A set of per-rank C2C plans replayed on one GPU (flagcxLocalPlan*)."""

    def __init__(self, cluster_ids, total_count, comm_op, red_op, is_inter=None):
        n = len(cluster_ids)
        self.nranks = n
        self._h = C.c_void_p()
        cl = (C.c_int * n)(*cluster_ids)
        it = (C.c_int * n)(*is_inter) if is_inter is not None else None
        rc = lib().flagcxLocalPlanCreate(C.byref(self._h), n, cl, it, total_count, int(comm_op), int(red_op))
        if rc:
            raise FlagcxError(rc, "flagcxLocalPlanCreate")

    def _check(self, rc):
        if rc:
            raise FlagcxError(rc, lib().flagcxLocalPlanGetLastError(self._h).decode() or
                              lib().flagcxLocalGetLastError().decode())

    def import_xml(self, prefix):
        self._check(lib().flagcxLocalPlanImportXml(self._h, prefix.encode()))

    def export_xml(self, prefix):
        self._check(lib().flagcxLocalPlanExportXml(self._h, prefix.encode()))

    def set_chunks(self, nchunks):
        self._check(lib().flagcxLocalPlanSetChunks(self._h, nchunks))

    def set_alltoallv(self, send_counts, s_displs, recv_counts, r_displs):
        """Four nranks x nranks matrices (nested lists), row r = rank r's arrays, in elements."""
        def flat(m):
            if m is None:
                return None
            v = [int(x) for row in m for x in row]
            return (C.c_size_t * len(v))(*v)
        self._check(lib().flagcxLocalPlanSetAlltoAllv(self._h, flat(send_counts), flat(s_displs), flat(recv_counts),
                                                      flat(r_displs)))

    def set_algorithm(self, algo):
        self._check(lib().flagcxLocalPlanSetAlgorithm(self._h, algo))

    def set_fused(self, fused):
        """True (default): refreshes are recorded and sums skip the cleared members; False: literal replay."""
        self._check(lib().flagcxLocalPlanSetFused(self._h, 1 if fused else 0))

    def traffic(self):
        """(algorithmic bytes, kernel launches) of the last execute."""
        b, n = C.c_uint64(), C.c_uint64()
        self._check(lib().flagcxLocalPlanGetTraffic(self._h, C.byref(b), C.byref(n)))
        return b.value, n.value

    def execute(self, send_ptrs, recv_ptrs, scratch_ptrs, dtype, root=-1, stream="current"):
        st = current_stream() if stream == "current" else stream
        sc = _ptr_array(scratch_ptrs) if scratch_ptrs is not None else None
        self._check(lib().flagcxLocalPlanExecute(self._h, _ptr_array(send_ptrs), _ptr_array(recv_ptrs), sc,
                                                 int(dtype), root, _sref(st)))

    def close(self):
        if self._h:
            lib().flagcxLocalPlanDestroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Ring:
    """Staging ring over caller memory (flagcxLocalRing*); ring_tensor stays referenced."""

    def __init__(self, ring_tensor, npeers, chunkbytes=0, steps=0):
        self._keep = ring_tensor
        self._h = C.c_void_p()
        rc = lib().flagcxLocalRingCreate(C.byref(self._h), ring_tensor.data_ptr(),
                                         ring_tensor.numel() * ring_tensor.element_size(), npeers, chunkbytes, steps)
        if rc:
            raise FlagcxError(rc, "flagcxLocalRingCreate")

    def send_recv(self, dst_ptr, src_ptr, size, copy_stream, stream):
        check(lib().flagcxLocalRingSendRecv(self._h, dst_ptr, src_ptr, size, C.byref(copy_stream), C.byref(stream)))

    def reduce_scatter(self, sendbuffs, rank, recv, op, copy_stream, stream, dtype=None):
        dt = dtype_of(recv, dtype)
        check(lib().flagcxLocalRingReduceScatter(self._h, _ptr_array([s.data_ptr() for s in sendbuffs]),
                                                 len(sendbuffs), rank, recv.data_ptr(), recv.numel(), int(dt),
                                                 int(op), C.byref(copy_stream), C.byref(stream)))

    def reduce_scatter_fifo(self, fifo, sendbuffs, rank, recv, copy_stream):
        """Proxy-style: staging copies on copy_stream, reduces through the running ReduceFifo; blocks."""
        rc = lib().flagcxLocalRingReduceScatterFifo(self._h, fifo._h, _ptr_array([s.data_ptr() for s in sendbuffs]),
                                                    len(sendbuffs), rank, recv.data_ptr(), recv.numel(),
                                                    C.byref(copy_stream))
        if rc:
            raise FlagcxError(rc, (lib().flagcxLocalReduceFifoGetLastError(fifo._h) or b"").decode())

    def close(self):
        if self._h:
            lib().flagcxLocalRingDestroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Gate:
    """A count that the host raises as the inputs of a gated batch complete (flagcxLocalGate*)."""

    def __init__(self):
        self._h = C.c_void_p()
        check(lib().flagcxLocalGateCreate(C.byref(self._h)))

    def reduce_batch(self, descs, op, dtype, nranks, stream="current"):
        """descs as reduce_batch; launched now, folded as open() passes each descriptor's number.
        Returns the number of descs[0]."""
        st = current_stream() if stream == "current" else stream
        keep = [_ptr_array(list(d[0])) for d in descs]
        arr = (ReduceDesc * len(descs))(*[ReduceDesc(keep[i], d[1], d[2]) for i, d in enumerate(descs)])
        first = C.c_uint64()
        check(lib().flagcxLocalReduceBatchGated(self._h, arr, len(descs), nranks, int(dtype), int(op), _sref(st),
                                                C.byref(first)))
        return first.value

    def open(self, upto):
        check(lib().flagcxLocalGateOpen(self._h, upto))

    def own_stream(self):
        """The gate's stream (a Stream structure): a hardware queue that nothing else shares."""
        p = C.POINTER(Stream)()
        check(lib().flagcxLocalGateOwnStream(self._h, C.byref(p)))
        return p.contents

    def query(self):
        """(descriptors numbered so far, count, state)."""
        a, b, st = C.c_uint64(), C.c_uint64(), C.c_int()
        check(lib().flagcxLocalGateQuery(self._h, C.byref(a), C.byref(b), C.byref(st)))
        return a.value, b.value, st.value

    def destroy(self):
        if self._h:
            h, self._h = self._h, C.c_void_p()
            check(lib().flagcxLocalGateDestroy(h))

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.destroy()
        return False


class ReduceFifo:
    """Host-producer / device-consumer reduce queue (flagcxLocalReduceFifo*).

    The consumer kernel is on the GPU while entries are outstanding and for a short linger
    after; then it parks and the next entry launches it again.  Use the object as a context
    manager so that an exception between start and stop still stops it.
    """

    def __init__(self, capacity, max_ranks, dtype, op):
        self._h = C.c_void_p()
        rc = lib().flagcxLocalReduceFifoCreate(C.byref(self._h), capacity, max_ranks, int(dtype), int(op))
        if rc:
            raise FlagcxError(rc, "flagcxLocalReduceFifoCreate")

    def _check(self, rc):
        if rc:
            raise FlagcxError(rc, (lib().flagcxLocalReduceFifoGetLastError(self._h) or b"").decode())

    def start(self):
        self._check(lib().flagcxLocalReduceFifoStart(self._h))
        return self

    def stop(self):
        self._check(lib().flagcxLocalReduceFifoStop(self._h))

    def try_enqueue_reduce(self, src_ptrs, dst_ptr, count):
        """Ticket, or None when the ring is full."""
        t = C.c_uint64()
        rc = lib().flagcxLocalReduceFifoEnqueueReduce(self._h, _ptr_array(src_ptrs), len(src_ptrs), dst_ptr, count,
                                                      C.byref(t))
        if rc == Result.InProgress:
            return None
        self._check(rc)
        return t.value

    def enqueue_reduce(self, src_ptrs, dst_ptr, count):
        while True:
            t = self.try_enqueue_reduce(src_ptrs, dst_ptr, count)
            if t is not None:
                return t

    def enqueue(self, trigger):
        t = C.c_uint64()
        while True:
            rc = lib().flagcxLocalReduceFifoEnqueue(self._h, C.byref(trigger), C.byref(t))
            if rc != Result.InProgress:
                break
        self._check(rc)
        return t.value

    def query(self):
        """(produced, consumed, state)"""
        p, c, st = C.c_uint64(), C.c_uint64(), C.c_int()
        self._check(lib().flagcxLocalReduceFifoQuery(self._h, C.byref(p), C.byref(c), C.byref(st)))
        return p.value, c.value, st.value

    def wait(self, ticket):
        self._check(lib().flagcxLocalReduceFifoWait(self._h, ticket))

    def set_window(self, nbytes):
        self._check(lib().flagcxLocalReduceFifoSetWindow(self._h, nbytes))

    def set_own_queue(self, own=True):
        """A hardware queue of its own for the consumer (its stream then is a blocking one)."""
        self._check(lib().flagcxLocalReduceFifoSetOwnQueue(self._h, 1 if own else 0))

    def set_linger(self, polls):
        self._check(lib().flagcxLocalReduceFifoSetLinger(self._h, polls))

    def set_waves(self, waves_per_cu):
        self._check(lib().flagcxLocalReduceFifoSetWaves(self._h, waves_per_cu))

    def grid(self):
        g = C.c_uint()
        self._check(lib().flagcxLocalReduceFifoGetGrid(self._h, C.byref(g)))
        return g.value

    def close(self):
        if self._h:
            lib().flagcxLocalReduceFifoDestroy(self._h)
            self._h = C.c_void_p()

    def __enter__(self):
        return self.start()

    def __exit__(self, *exc):
        try:
            lib().flagcxLocalReduceFifoStop(self._h)
        finally:
            return False

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


ADAPTOR_SLOTS = [
    "deviceSynchronize", "deviceMemcpy", "deviceMemset", "deviceMalloc", "deviceFree", "setDevice", "getDevice",
    "getDeviceCount", "getVendor", "hostGetDevicePointer", "memHandleInit", "memHandleDestroy", "gdrMemAlloc",
    "gdrMemFree", "hostShareMemAlloc", "hostShareMemFree", "gdrPtrMmap", "gdrPtrMunmap", "streamCreate",
    "streamDestroy", "streamCopy", "streamFree", "streamSynchronize", "streamQuery", "streamWaitEvent",
    "eventCreate", "eventDestroy", "eventRecord", "eventSynchronize", "eventQuery", "ipcMemHandleCreate",
    "ipcMemHandleGet", "ipcMemHandleOpen", "ipcMemHandleClose", "ipcMemHandleFree", "launchKernel", "copyArgsInit",
    "copyArgsFree", "launchDeviceFunc", "getDeviceProperties", "getDevicePciBusId", "getDeviceByPciBusId",
    "launchHostFunc", "dmaSupport", "getHandleForAddressRange", "eventElapsedTime",
]


def device_adaptor():
    """(name, {slot: address or None}) of the exported flagcxDeviceAdaptor table."""
    base = lib().flagcxLocalGetDeviceAdaptor()
    name = C.string_at(base, 32).split(b"\0")[0].decode()
    ptrs = (C.c_void_p * len(ADAPTOR_SLOTS)).from_address(base + 32)
    return name, {n: ptrs[k] for k, n in enumerate(ADAPTOR_SLOTS)}


def adaptor_fn(slots, name, restype, *argtypes):
    return C.CFUNCTYPE(restype, *argtypes)(slots[name])

"""KvCache: the key / value caches of several sequences over the C ABI (qph_kv_*), for torch tensors on the GPU.

Calls go to the current stream of the tensors' device and are not waited for; they can be captured into a graph, which then
reads pos and lens anew at every replay."""
import ctypes as C

from ._lib import QPH_F16, QPH_Q4, QphError, check, lib

_KINDS = {"f16": QPH_F16, "q4": QPH_Q4, QPH_F16: QPH_F16, QPH_Q4: QPH_Q4}
_bind = None


def _binding():
    """the compiled half of this file (csrc/kvbind.cpp), told what it uses of torch's Python side"""
    global _bind
    if _bind is None:
        import torch
        lib()   # the library, with its message where it has not been built
        try:
            from . import _kvbind
        except ImportError as e:
            raise QphError(f"kv: the compiled binding (_kvbind.so) was not built, or for another torch than {torch.__version__}: run make in qpack_amd/csrc ({e})") from e
        _kvbind.setup(QphError, torch._C._cuda_getCurrentRawStream, torch.cuda.current_device, torch.cuda.device)
        _bind = _kvbind
    return _bind


def _strides(x):
    """between the sequences and positions of an f16 cache's tensor; 0 (without gaps) for an axis of one, whose stride means nothing"""
    return tuple(stride if size > 1 else 0 for size, stride in zip(x.shape[:2], x.stride()))


class KvCache:
    """nseq sequences of ctx positions, kv_heads heads of head_dim (64 or 128) dims, in fp16 ("f16") or 4 bits ("q4").

    data: the memory, new (zeros) when None.  "q4": a contiguous uint8 tensor [nseq, kv_heads, ceil(ctx / 8), 9 * head_dim] of
    the records that include/qpack_hip.h describes; "f16": (K, V), fp16 tensors [nseq, ctx, kv_heads, head_dim] of equal strides, each
    position's rows contiguous, sequences and positions apart (no expanded tensors).

    In all calls token t < n of sequence b, and t < lens[b] where lens is given, is position pos[b] + t; sequences with pos[b] <
    0 and positions at or past ctx take no part.  pos and lens: int32 tensors [nseq] on the cache's device.

    Writes to one cache follow each other: from several streams they need events between them.  Nothing here carries
    gradients: tensors that require one are refused while gradients are recorded."""

    def __init__(self, kind, nseq, kv_heads, head_dim, ctx, data=None, device="cuda"):
        import torch
        if kind not in _KINDS:
            raise QphError(f"kv: kind must be 'f16' or 'q4', not {kind!r}")
        self.kind, self.nseq, self.kv_heads, self.head_dim, self.ctx = _KINDS[kind], int(nseq), int(kv_heads), int(head_dim), int(ctx)
        b = C.c_int64()
        check(lib().qph_kv_bytes(self.kind, self.nseq, self.kv_heads, self.head_dim, self.ctx, C.byref(b)))
        self.nbytes = b.value
        if self.kind == QPH_Q4:
            shape = (self.nseq, self.kv_heads, (self.ctx + 7) // 8, 9 * self.head_dim)
            if data is None:
                data = torch.zeros(shape, dtype=torch.uint8, device=device)
            if data.dtype != torch.uint8 or tuple(data.shape) != shape or not data.is_contiguous():
                raise QphError(f"kv: a q4 cache's data must be a contiguous uint8 tensor {list(shape)}")
            tensors, at = (data,), (data.data_ptr(), 0, 0, 0)
        else:
            shape = (self.nseq, self.ctx, self.kv_heads, self.head_dim)
            if data is None:
                data = tuple(torch.zeros(shape, dtype=torch.float16, device=device) for _ in range(2))
            k, v = data
            for x in (k, v):
                if x.dtype != torch.float16 or tuple(x.shape) != shape or x.stride(3) != 1 or (self.kv_heads > 1 and x.stride(2) != self.head_dim) or _strides(x) != _strides(k):
                    raise QphError(f"kv: an f16 cache's data must be two fp16 tensors {list(shape)} of equal strides with contiguous rows")
                if any(size > 1 and stride == 0 for size, stride in zip(x.shape[:2], x.stride())):
                    raise QphError("kv: an f16 cache's sequences and positions must not share memory (an expanded tensor)")
            if v.device != k.device:
                raise QphError("kv: K and V on different devices")
            tensors, at = (k, v), (k.data_ptr(), v.data_ptr(), *_strides(k))
        if torch.is_grad_enabled() and any(x.requires_grad for x in tensors):
            raise QphError("kv: the cache's data requires a gradient, and no call here passes one on")
        first = tensors[0]
        if first.device.type != "cuda":
            raise QphError("kv: the cache must be on a GPU")
        self.data, self.device = data, first.device
        self._c = _binding().Cache(self.kind, self.nseq, self.kv_heads, self.head_dim, self.ctx, *at, self.device.index, *tensors)

    def write(self, k, v, pos, lens=None):
        """round the rows k and v [nseq, n, kv_heads, head_dim] into the cache"""
        self._c.write(k, v, pos, lens)

    def read(self, pos, n, dtype=None, lens=None, out=None):
        """(k, v) [nseq, n, kv_heads, head_dim]: what the cache holds, in dtype (float16 when None); into out = (k, v) where given.  Rows
        that take no part stay as they are in out, and are zero without it"""
        if out is None:
            import torch
            shape = (self.nseq, int(n), self.kv_heads, self.head_dim)
            out = tuple(torch.zeros(shape, dtype=dtype or torch.float16, device=self.device) for _ in range(2))
        k, v = out
        if k.shape[1] != n:
            raise QphError("kv: out must have n tokens")
        self._c.read(k, v, pos, lens)
        return out

    def attention(self, q, pos, lens=None, window=0, sinks=0, scale=0.0, out=None):
        """softmax(scale q K^T) V of the tokens q [nseq, n, heads, head_dim] at pos[b] + t, whose rows are in the cache; scale 0: 1 /
        sqrt(head_dim).  Position P sees p <= P and, with window > 0, of those p > P - window and p < sinks only.  out may be q, or apart from it; rows that
        take no part stay as they are in out, and are zero without it"""
        if out is None:
            import torch
            out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        self._c.attention(q, out, pos, lens, window, sinks, scale)
        return out

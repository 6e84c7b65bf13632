"""KvCache: the key / value caches of several sequences over the C ABI (qph_kv_*), for torch tensors on the GPU.

Calls go to the current stream of the tensors' device and are not waited for; they can be captured into a graph, which then
reads pos and lens anew at every replay."""
import ctypes as C

from ._lib import QPH_BF16, QPH_F16, QPH_F32, QPH_Q4, KvC, QphError, RowsC, check, lib

_KINDS = {"f16": QPH_F16, "q4": QPH_Q4, QPH_F16: QPH_F16, QPH_Q4: QPH_Q4}
_TYPES = {}


def _types():
    if not _TYPES:
        import torch
        _TYPES.update({torch.float32: QPH_F32, torch.float16: QPH_F16, torch.bfloat16: QPH_BF16})
    return _TYPES


class KvCache:
    """nseq sequences of ctx positions, kv_heads heads of head_dim (64 or 128) dims, in fp16 ("f16") or 4 bits ("q4").

    data: the memory, new (zeros) when None.  "q4": a contiguous uint8 tensor [nseq, kv_heads, ceil(ctx / 8), 9 * head_dim] of
    the records that include/qpack_hip.h describes; "f16": (K, V), fp16 tensors [nseq, ctx, kv_heads, head_dim] of equal strides, each
    position's rows contiguous.

    In all calls token t < n of sequence b, and t < lens[b] where lens is given, is position pos[b] + t; sequences with pos[b] <
    0 and positions at or past ctx take no part.  pos and lens: int32 tensors [nseq] on the cache's device."""

    def __init__(self, kind, nseq, kv_heads, head_dim, ctx, data=None, device="cuda"):
        import torch
        if kind not in _KINDS:
            raise QphError(f"kv: kind must be 'f16' or 'q4', not {kind!r}")
        self.kind, self.nseq, self.kv_heads, self.head_dim, self.ctx = _KINDS[kind], int(nseq), int(kv_heads), int(head_dim), int(ctx)
        b = C.c_int64()
        check(lib().qph_kv_bytes(self.kind, self.nseq, self.kv_heads, self.head_dim, self.ctx, C.byref(b)))
        self.nbytes = b.value
        c = KvC(self.kind, self.nseq, self.kv_heads, self.head_dim, self.ctx)
        if self.kind == QPH_Q4:
            shape = (self.nseq, self.kv_heads, (self.ctx + 7) // 8, 9 * self.head_dim)
            if data is None:
                data = torch.zeros(shape, dtype=torch.uint8, device=device)
            if data.dtype != torch.uint8 or tuple(data.shape) != shape or not data.is_contiguous():
                raise QphError(f"kv: a q4 cache's data must be a contiguous uint8 tensor {list(shape)}")
            first = data
            c.k = data.data_ptr()
        else:
            shape = (self.nseq, self.ctx, self.kv_heads, self.head_dim)
            if data is None:
                data = tuple(torch.zeros(shape, dtype=torch.float16, device=device) for _ in range(2))
            k, v = data
            for x in (k, v):
                if x.dtype != torch.float16 or tuple(x.shape) != shape or x.stride()[2:] != (self.head_dim, 1) or x.stride() != k.stride():
                    raise QphError(f"kv: an f16 cache's data must be two fp16 tensors {list(shape)} of equal strides with contiguous rows")
            if v.device != k.device:
                raise QphError("kv: K and V on different devices")
            first = k
            c.k, c.v, c.seq, c.row = k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1)
        if first.device.type != "cuda":
            raise QphError("kv: the cache must be on a GPU")
        self.data, self.device, self._c = data, first.device, c
        self._ref = C.byref(c)
        self._work = {}

    def _rows(self, x, name, heads=None):
        t = _types().get(x.dtype)
        if t is None:
            raise QphError(f"kv: {name} must be float32, float16 or bfloat16, not {x.dtype}")
        if x.device != self.device:
            raise QphError(f"kv: {name} is on {x.device}, the cache on {self.device}")
        s, st = x.shape, x.stride()
        if len(s) != 4 or s[0] != self.nseq or s[3] != self.head_dim or (heads is not None and s[2] != heads):
            raise QphError(f"kv: {name} must be [{self.nseq}, n, {heads or 'heads'}, {self.head_dim}], not {list(s)}")
        if st[3] != 1:
            raise QphError(f"kv: the last dimension of {name} must be contiguous")
        return RowsC(x.data_ptr(), t, st[0], st[1], st[2])

    def _index(self, x, name):
        import torch
        if x is None and name == "lens":
            return None
        if x.dtype != torch.int32 or x.device != self.device or tuple(x.shape) != (self.nseq,) or not x.is_contiguous():
            raise QphError(f"kv: {name} must be a contiguous int32 tensor [{self.nseq}] on {self.device}")
        return x.data_ptr()

    def _run(self, f, *args):
        import torch
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return check(f(*args, torch.cuda.current_stream().cuda_stream))
        check(f(*args, torch.cuda.current_stream().cuda_stream))

    def write(self, k, v, pos, lens=None):
        """round the rows k and v [nseq, n, kv_heads, head_dim] into the cache"""
        rk, rv = self._rows(k, "k", self.kv_heads), self._rows(v, "v", self.kv_heads)
        if k.shape[1] != v.shape[1]:
            raise QphError("kv: k and v have different numbers of tokens")
        self._run(lib().qph_kv_write, self._ref, C.byref(rk), C.byref(rv), k.shape[1], self._index(pos, "pos"), self._index(lens, "lens"))

    def read(self, pos, n, dtype=None, lens=None, out=None):
        """(k, v) [nseq, n, kv_heads, head_dim]: what the cache holds, in dtype (float16 when None); into out = (k, v) where given.  Rows
        that take no part stay as they are in out, and are zero without it"""
        import torch
        if out is None:
            shape = (self.nseq, int(n), self.kv_heads, self.head_dim)
            out = tuple(torch.zeros(shape, dtype=dtype or torch.float16, device=self.device) for _ in range(2))
        k, v = out
        rk, rv = self._rows(k, "k", self.kv_heads), self._rows(v, "v", self.kv_heads)
        if k.shape[1] != n or v.shape[1] != n:
            raise QphError("kv: out must have n tokens")
        self._run(lib().qph_kv_read, self._ref, C.byref(rk), C.byref(rv), int(n), self._index(pos, "pos"), self._index(lens, "lens"))
        return out

    def attention(self, q, pos, lens=None, window=0, sinks=0, scale=0.0, out=None):
        """softmax(scale q K^T) V of the tokens q [nseq, n, heads, head_dim] at pos[b] + t, whose rows are in the cache; scale 0: 1 /
        sqrt(head_dim).  Position P sees p <= P and, with window > 0, of those p > P - window and p < sinks only.  out may be q; rows that
        take no part stay as they are in out, and are zero without it"""
        import torch
        if out is None:
            out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        rq, ro = self._rows(q, "q"), self._rows(out, "out")
        n, heads = q.shape[1], q.shape[2]
        if out.shape != q.shape:
            raise QphError("kv: out must have q's shape")
        key = (rq.type, heads, n, window, sinks)
        size = self._work.get(key)   # sizes alone are kept: the scratch is each call's own
        if size is None:
            b = C.c_int64()
            check(lib().qph_kv_attention_work(self._ref, rq.type, heads, n, window, sinks, C.byref(b)))
            size = self._work[key] = b.value
        work = torch.empty(size, dtype=torch.uint8, device=self.device) if size else None
        self._run(lib().qph_kv_attention, self._ref, C.byref(rq), C.byref(ro), heads, n, self._index(pos, "pos"), self._index(lens, "lens"),
                  window, sinks, scale, work.data_ptr() if size else None, size)
        return out

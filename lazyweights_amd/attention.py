"""Attention between a decoder layer's coded matrices, on torch tensors: a paged key-value cache, a batch of sequences over
it, and the operators of include/lazyweights_amd.h that append to the cache and read it (lw_kv_append, lw_attn_decode,
lw_attn_prompt; lw_kv8_append, lw_attn8_decode, lw_attn8_prompt over a cache held in 8 bits). lazyweights_amd/pages.py makes
q_start, kv_len and page_table on the GPU.

    cache = KvCache.empty(pages, kv_heads, page_size, head_dim)          # one per layer; or KvCache8, of half the size
    batch = Batch(cache, heads, q_start, kv_len, page_table, max_new, max_kv)  # one for all layers
    q16 = cache.append(batch, q, k, v, cos, sin)                         # q, k, v as the matrices give them, fp32
    y = cache.attend_decode(batch, q16)                                  # or attend_prompt, for more than 16 new tokens

The tensors of a batch (q_start, kv_len, page_table) are read on the GPU when a call runs: a program that writes the next
step's lengths and pages into them keeps the batch, and can capture its calls, as long as max_new and max_kv bound them.
Calls go to torch's current stream unless `stream` (a hipStream_t as an integer) is given. Then what a call returns belongs to
that stream, and the memory of what it reads is not given to others before the call is done (torch's record_stream: a stream
of the caller's own has to outlive these tensors); that the given stream waits for what made the inputs (a Batch fills its
workspace on the stream that is current when it is made) is the caller's part, as with all of torch. Bad arguments raise
ValueError; a call that the library refuses raises RuntimeError with lw_last_error().
"""
import ctypes

try:
    import torch
except ImportError:  # (bundles and the host entry points need none)
    torch = None

from ._lib import last_error, load_library

F32, F16, BF16 = 0, 1, 2


class _Cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("pages", ctypes.c_int64),
                ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("row_stride", ctypes.c_int64),
                ("page_size", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("type", ctypes.c_int32)]


class _Batch(ctypes.Structure):
    _fields_ = [("seqs", ctypes.c_int32), ("tokens", ctypes.c_int32), ("max_new", ctypes.c_int32),
                ("max_kv", ctypes.c_int32), ("q_start", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("page_table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("table_pages", ctypes.c_int32),
                ("reserved", ctypes.c_int32), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_int64)]


def _types():
    return {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def _current_stream():
    """A function: device index -> torch's current stream there, as an integer."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # a tenth of the public call's 2 us
    return raw or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _current_device():
    """A function: the index of torch's current device."""
    return getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _Cache8(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_exp", ctypes.c_void_p), ("v_exp", ctypes.c_void_p),
                ("pages", ctypes.c_int64), ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("row_stride", ctypes.c_int64), ("exp_page_stride", ctypes.c_int64), ("exp_head_stride", ctypes.c_int64),
                ("page_size", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("reserved", ctypes.c_int32)]


class Batch:
    """`seqs` sequences whose new tokens are the rows of a call: q_start int32 [seqs + 1], kv_len int32 [seqs] (the lengths
    with the new tokens), page_table int32 [seqs, pages], all on the cache's GPU. max_new and max_kv bound every
    sequence's new tokens and length. A call's tensors may have more rows than q_start names; those are left alone. Holds
    the workspace of attend_decode and attend_prompt, so calls with one batch must not overlap. It serves every cache on its
    device whose page tables are the same (all layers of a model); with max_new <= 16 attention is for caches of as many
    key-value heads as the one it was made for, and as it in 16 or in 8 bits, since the workspace's counters are laid out by
    them."""

    def __init__(self, cache, heads, q_start, kv_len, page_table, max_new, max_kv):
        seqs = kv_len.shape[0]
        if q_start.shape != (seqs + 1,) or kv_len.dim() != 1 or page_table.dim() != 2 or page_table.shape[0] != seqs:
            raise ValueError("q_start [seqs + 1], kv_len [seqs] and page_table [seqs, pages] are wanted, not %s, %s, %s"
                             % (tuple(q_start.shape), tuple(kv_len.shape), tuple(page_table.shape)))
        for t in (q_start, kv_len, page_table):
            if t.dtype != torch.int32 or t.device != cache.k.device:
                raise ValueError("q_start, kv_len and page_table must be int32 tensors on the cache's device")
            if t.numel() and t.stride(-1) != 1:
                raise ValueError("q_start, kv_len and the rows of page_table must be contiguous")
        self.heads, self.max_new, self.max_kv = int(heads), int(max_new), int(max_kv)
        if not all(-1 << 31 <= n < 1 << 31 for n in (self.heads, self.max_new, self.max_kv)):
            raise ValueError("heads, max_new and max_kv must be numbers of 32 bits")  # (others would be cut to that)
        self.tensors = (q_start, kv_len, page_table)  # kept alive
        self.index, self.kv_heads, self.eight = cache.index, cache.kv_heads, cache.eight
        self.c = _Batch(seqs, 0, self.max_new, self.max_kv, q_start.data_ptr(), kv_len.data_ptr(),
                        page_table.data_ptr(), page_table.stride(0) if seqs > 1 else page_table.shape[1],
                        page_table.shape[1], 0, None, 0)
        self.ptr = ctypes.addressof(self.c)
        size = cache._workspace_size(self)
        if size < 0:
            raise ValueError(last_error())
        self.workspace = torch.zeros(size, dtype=torch.uint8, device=cache.k.device)
        self.c.workspace, self.c.workspace_bytes = self.workspace.data_ptr(), size


class KvCache:
    """Keys and values [pages, kv_heads, page_size, head_dim] of one layer, float16 or bfloat16 on the GPU, the caller's
    tensors or views of them with head_dim contiguous (k and v alike in their strides)."""

    eight = False

    def __init__(self, k, v):
        types = _types()
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.stride() != v.stride():
            raise ValueError("k and v must be [pages, kv_heads, page_size, head_dim], alike in type, device and strides")
        if not k.is_cuda or types.get(k.dtype) not in (F16, BF16):
            raise ValueError("k and v must be float16 or bfloat16 tensors on the GPU")
        if k.stride(3) != 1:
            raise ValueError("the elements of a head must be contiguous")
        self.lib, self.k, self.v = load_library(), k, v
        self.kv_heads, self.head_dim = k.shape[1], k.shape[3]
        self.types, self.index = types, k.get_device()
        self._current, self._device = _current_stream(), _current_device()
        self.c = _Cache(k.data_ptr(), v.data_ptr(), k.shape[0], k.stride(0), k.stride(1), k.stride(2), k.shape[2],
                        k.shape[1], k.shape[3], types[k.dtype])
        self.ptr = ctypes.addressof(self.c)

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, dtype=None, device="cuda"):
        """A new cache of float16 (or `dtype`); its contents are whatever the memory held."""
        k, v = (torch.empty((pages, kv_heads, page_size, head_dim), dtype=dtype or torch.float16, device=device)
                for _ in range(2))
        return cls(k, v)

    def _workspace_size(self, batch):
        return self.lib.lw_attn_workspace(self.ptr, batch.ptr, batch.heads)

    def _memory(self):
        return self.k, self.v

    def _rows(self, what, x, heads):
        """Rows, address and row stride of x [tokens, heads, head_dim] or [tokens, heads * head_dim]."""
        shape, stride, dim = x.shape, x.stride(), self.head_dim
        if len(shape) == 3:
            ok = shape[1] == heads and shape[2] == dim and stride[2] == 1 and (heads == 1 or stride[1] == dim)
        else:
            ok = len(shape) == 2 and shape[1] == heads * dim and stride[1] == 1
        if not ok or x.get_device() != self.index:
            raise ValueError("%s: [tokens, %d, %d] (or the two last joined) with contiguous rows on the cache's device is "
                             "wanted, not %s" % (what, heads, dim, tuple(shape)))
        rows = shape[0]
        return rows, x.data_ptr(), stride[0] if rows > 1 else heads * dim

    def _other(self, stream):
        """torch's stream of the handle `stream`; None if that is the current one."""
        if stream == self._current(self.index):
            return None
        return torch.cuda.ExternalStream(stream, self.index) if stream else torch.cuda.default_stream(self.index)

    def _empty(self, shape, dtype, other):
        """A new tensor of the memory of the stream that is going to write it."""
        if other is None:
            return torch.empty(shape, dtype=dtype, device=self.k.device)
        with torch.cuda.stream(other):
            return torch.empty(shape, dtype=dtype, device=self.k.device)

    def _used(self, other, batch, *tensors):
        """Keeps the memory of a call's tensors from others until the stream `other` has done the call."""
        for t in self._memory() + (batch.workspace,) + batch.tensors + tensors:
            if t is not None:
                t.record_stream(other)

    def append(self, batch, q, k, v, cos=None, sin=None, q_out=None, neighbours=False, stream=None):
        """Appends the rows k, v [tokens, kv_heads, head_dim] of the batch's new tokens, k rotated by its position, and
        returns q [tokens, heads, head_dim], rotated alike, in the cache's type (q may be None: keys and values only).
        q, k and v have one type (float32, float16 or bfloat16); rows may be views into a joined projection. cos, sin
        float32 [positions, rot / 2] rotate the first rot elements of a head in pairs (j, j + rot / 2), or (2 j, 2 j + 1)
        with `neighbours`; without them nothing is rotated."""
        if self._device() != self.index:  # launches go to the current device
            with torch.cuda.device(self.index):
                return self.append(batch, q, k, v, cos, sin, q_out, neighbours, stream)
        if batch.index != self.index:
            raise ValueError("the batch is on another device than the cache")
        heads, dtype = batch.heads, k.dtype
        kind = self.types.get(dtype)
        n, kp, ldk = self._rows("k", k, self.kv_heads)
        nv, vp, ldv = self._rows("v", v, self.kv_heads)
        nq, qp, ldq = (n, None, 0) if q is None else self._rows("q", q, heads)
        if kind is None or v.dtype != dtype or nv != n or nq != n or (q is not None and q.dtype != dtype):
            raise ValueError("q, k and v must have one of the types float32, float16, bfloat16 and the same number of rows")
        other = None if stream is None else self._other(stream)
        op, ldo, q_dtype = None, 0, None
        if q is not None:
            q_dtype = self._q_dtype(q_out) if self.eight else self.k.dtype
            if q_out is None:
                q_out = self._empty((n, heads, self.head_dim), q_dtype, other)
            no, op, ldo = self._rows("q_out", q_out, heads)
            if q_out.dtype != q_dtype or no != n:
                raise ValueError("q_out must have the cache's type and q's rows")
        cp, sp, rot, rows = None, None, 0, 0
        if cos is not None or sin is not None:
            shape = () if cos is None else cos.shape
            if (sin is None or len(shape) != 2 or cos.dtype != torch.float32 or sin.dtype != torch.float32
                    or shape != sin.shape or cos.get_device() != self.index or sin.get_device() != self.index
                    or not cos.is_contiguous() or not sin.is_contiguous()):
                raise ValueError("cos and sin must be contiguous float32 tensors [positions, rot / 2] on the cache's device")
            rows, rot = shape
            cp, sp, rows, rot = cos.data_ptr(), sin.data_ptr(), min(rows, (1 << 31) - 1), 2 * rot
        batch.c.tokens = n
        where = self._current(self.index) if stream is None else stream
        if self.eight:
            rc = self.lib.lw_kv8_append(self.ptr, batch.ptr, heads, qp, kp, vp, kind, ldq, ldk, ldv, cp, sp, rot, rows,
                                        1 if neighbours else 0, op, F16 if q is None else self.types[q_dtype], ldo, where)
        else:
            rc = self.lib.lw_kv_append(self.ptr, batch.ptr, heads, qp, kp, vp, kind, ldq, ldk, ldv, cp, sp, rot, rows,
                                       1 if neighbours else 0, op, ldo, where)
        if rc != 0:
            raise RuntimeError(last_error())
        if other is not None:
            self._used(other, batch, q, k, v, cos, sin, q_out)
        return q_out

    def _attend(self, call, batch, q, out, scale, window, stream):
        if self._device() != self.index:  # launches go to the current device
            with torch.cuda.device(self.index):
                return self._attend(call, batch, q, out, scale, window, stream)
        heads = batch.heads
        if batch.index != self.index:
            raise ValueError("the batch is on another device than the cache")
        if batch.kv_heads != self.kv_heads and batch.max_new <= 16:
            raise ValueError("the batch is for caches of %d key-value heads, not %d" % (batch.kv_heads, self.kv_heads))
        if batch.eight != self.eight and batch.max_new <= 16:
            raise ValueError("the batch is for caches in %d bits" % (8 if batch.eight else 16))
        if not 0 <= window < 1 << 31:  # (32 bits in the call: no position is that far back)
            window = (1 << 31) - 1 if window > 0 else -1
        dtype = q.dtype
        if dtype != (self._q_type(dtype) if self.eight else self.k.dtype):
            raise ValueError("q must have the cache's type")
        n, qp, ldq = self._rows("q", q, heads)
        other = None if stream is None else self._other(stream)
        if out is None:
            out = self._empty(q.shape, dtype, other)
        kind = self.types.get(out.dtype)
        no, op, ldo = self._rows("out", out, heads)
        if kind is None or no != n:
            raise ValueError("out must be float32, float16 or bfloat16, with q's rows")
        batch.c.tokens = n
        scale, where = self.head_dim ** -0.5 if scale is None else scale, self._current(self.index) if stream is None else stream
        if self.eight:
            rc = call(self.ptr, batch.ptr, heads, qp, self.types[dtype], ldq, op, kind, ldo, scale, window, where)
        else:
            rc = call(self.ptr, batch.ptr, heads, qp, ldq, op, kind, ldo, scale, window, where)
        if rc != 0:
            raise RuntimeError(last_error())
        if other is not None:
            self._used(other, batch, q, out)
        return out

    def attend_decode(self, batch, q, out=None, scale=None, window=0, stream=None):
        """Attention of at most 16 new tokens per sequence over the cache, q [tokens, heads, head_dim] as append gives it:
        every row sees the positions up to its own (the last `window` of them if window > 0), weights
        softmax(scale q . k), scale 1 / sqrt(head_dim) by default. Returns out (q's type by default; float32, float16 and
        bfloat16 can be given). A row that sees nothing gives zeros."""
        return self._attend(self.lib.lw_attn_decode, batch, q, out, scale, window, stream)

    def attend_prompt(self, batch, q, out=None, scale=None, window=0, stream=None):
        """attend_decode for any number of new tokens: whole prompts, or chunks of them after what is in the cache."""
        return self._attend(self.lib.lw_attn_prompt, batch, q, out, scale, window, stream)


class KvCache8(KvCache):
    """Keys and values of one layer in 8 bits: k and v float8_e4m3fn [pages, kv_heads, page_size, head_dim] on the GPU (as
    KvCache's, page_size 16 at least), k_exp and v_exp int8 [pages, kv_heads, page_size / 16] with the last dimension
    contiguous and alike in their strides: an element is its number times two to the exponent of its 16 rows' block. append
    chooses the exponents (lw_kv8_append): the least that holds a block's new rows, and older rows of the block are rounded to a
    larger one where it grows. q is float16 or bfloat16: append gives `q_dtype`, or the type of q_out. A Batch serves
    caches of one kind only, of 8 or of 16 bits."""

    eight = True

    def __init__(self, k, v, k_exp, v_exp, q_dtype=None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.stride() != v.stride():
            raise ValueError("k and v must be [pages, kv_heads, page_size, head_dim], alike in type, device and strides")
        if not k.is_cuda or k.dtype != torch.float8_e4m3fn:
            raise ValueError("k and v must be float8_e4m3fn tensors on the GPU")
        if k.stride(3) != 1:
            raise ValueError("the elements of a head must be contiguous")
        want = (k.shape[0], k.shape[1], k.shape[2] // 16)
        if any(t.shape != want or t.dtype != torch.int8 or t.device != k.device for t in (k_exp, v_exp)):
            raise ValueError("k_exp and v_exp must be int8 tensors [pages, kv_heads, page_size / 16] on the cache's device")
        if k_exp.stride() != v_exp.stride() or (want[2] > 1 and k_exp.stride(2) != 1):
            raise ValueError("k_exp and v_exp must be alike in their strides, a head's exponents contiguous")
        self.lib, self.k, self.v, self.k_exp, self.v_exp = load_library(), k, v, k_exp, v_exp
        self.kv_heads, self.head_dim = k.shape[1], k.shape[3]
        self.types, self.index = _types(), k.get_device()
        self.q_dtype = self._q_type(q_dtype or torch.float16)
        self._current, self._device = _current_stream(), _current_device()
        self.c = _Cache8(k.data_ptr(), v.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), k.shape[0], k.stride(0), k.stride(1),
                         k.stride(2), k_exp.stride(0), k_exp.stride(1), k.shape[2], k.shape[1], k.shape[3], 0)
        self.ptr = ctypes.addressof(self.c)

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, q_dtype=None, device="cuda"):
        """A new cache; its contents are whatever the memory held."""
        k, v = (torch.empty((pages, kv_heads, page_size, head_dim), dtype=torch.float8_e4m3fn, device=device) for _ in range(2))
        k_exp, v_exp = (torch.empty((pages, kv_heads, page_size // 16), dtype=torch.int8, device=device) for _ in range(2))
        return cls(k, v, k_exp, v_exp, q_dtype)

    def _workspace_size(self, batch):
        return self.lib.lw_attn8_workspace(self.ptr, batch.ptr, batch.heads)

    def _memory(self):
        return self.k, self.v, self.k_exp, self.v_exp

    def _q_type(self, dtype):
        if self.types.get(dtype) not in (F16, BF16):
            raise ValueError("q over an 8-bit cache is float16 or bfloat16")
        return dtype

    def _q_dtype(self, q_out):
        """The type that q gets when it is appended, into q_out if that is given."""
        return self.q_dtype if q_out is None else self._q_type(q_out.dtype)

    def attend_decode(self, batch, q, out=None, scale=None, window=0, stream=None):
        """KvCache.attend_decode, q float16 or bfloat16."""
        return self._attend(self.lib.lw_attn8_decode, batch, q, out, scale, window, stream)

    def attend_prompt(self, batch, q, out=None, scale=None, window=0, stream=None):
        """KvCache.attend_prompt, q float16 or bfloat16."""
        return self._attend(self.lib.lw_attn8_prompt, batch, q, out, scale, window, stream)

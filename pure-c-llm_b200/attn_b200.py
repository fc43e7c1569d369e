"""ctypes binding of libattn_b200.so -- the host-side mirror of the C ABI
declared in include/attn_b200.h.

The names follow the reference's call surface (attn_fwd / attn_bwd of
gpu_kernels.h:67-72, cached_attention of transformer.c:203).  Raw-pointer
wrappers take integer device addresses; the `*_t` helpers take torch CUDA
tensors, which serve only as device memory and stream plumbing.  There is
no fallback: if the shared library is missing, importing this module raises.
"""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libattn_b200.so")

OK, ERR_INVALID, ERR_UNSUPPORTED, ERR_CUDA, ERR_NOMEM, ERR_WORKSPACE, ERR_DEVICE, ERR_COMM = range(8)
PROBS_LSE_OUT, PROBS_LSE = 0, 1      # attn_set_probs_mode
F32, BF16, I8 = 0, 1, 2
MAX_LAYERS = 64
ROPE_PLAIN, ROPE_LINEAR, ROPE_BASE, ROPE_RAMP = range(4)   # attn_rope_config.scaling
STATIC_SCRATCH_BYTES = 4 << 20      # ATTN_DECODE_STATIC_SCRATCH_BYTES


class AttnError(RuntimeError):
    def __init__(self, status, msg):
        super().__init__(f"attn status {status}: {msg}")
        self.status = status


if not os.path.exists(LIB_PATH):
    raise ImportError(f"{LIB_PATH} is not built; run `make -C pure-c-llm_b200` (or __graft_entry__.build())")
lib = ctypes.CDLL(LIB_PATH)


class Shape(ctypes.Structure):
    _fields_ = [("batch", ctypes.c_int), ("heads", ctypes.c_int), ("seq_len", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("in_row_stride", ctypes.c_longlong),
                ("out_row_stride", ctypes.c_longlong)]


class DecodeShape(ctypes.Structure):
    _fields_ = [("n_seq", ctypes.c_int), ("heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("kv_dtype", ctypes.c_int), ("row_stride", ctypes.c_longlong),
                ("cap", ctypes.c_longlong), ("max_len", ctypes.c_int)]


class KVCache(ctypes.Structure):
    _fields_ = [("n_layers", ctypes.c_int), ("cap", ctypes.c_int), ("heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("kv_dtype", ctypes.c_int),
                ("k", ctypes.c_void_p * MAX_LAYERS), ("v", ctypes.c_void_p * MAX_LAYERS),
                ("kscale", ctypes.c_void_p * MAX_LAYERS), ("vscale", ctypes.c_void_p * MAX_LAYERS)]


class QKVShape(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_int), ("in_features", ctypes.c_int), ("out_features", ctypes.c_int),
                ("x_row_stride", ctypes.c_longlong), ("out_row_stride", ctypes.c_longlong)]


class PagedKV(ctypes.Structure):
    _fields_ = [("kv_dtype", ctypes.c_int), ("rows", ctypes.c_longlong), ("row_stride", ctypes.c_longlong),
                ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("kscale", ctypes.c_void_p), ("vscale", ctypes.c_void_p)]


class PageShape(ctypes.Structure):
    _fields_ = [("n_seq", ctypes.c_int), ("page_size", ctypes.c_int), ("max_pages", ctypes.c_int),
                ("max_tokens", ctypes.c_int), ("n_pages", ctypes.c_int), ("table_stride", ctypes.c_int)]


class RopeConfig(ctypes.Structure):
    _fields_ = [("rot_dim", ctypes.c_int), ("max_pos", ctypes.c_int), ("scaling", ctypes.c_int),
                ("trained_len", ctypes.c_int), ("base", ctypes.c_double), ("factor", ctypes.c_double),
                ("fast", ctypes.c_double), ("slow", ctypes.c_double), ("magnitude", ctypes.c_double)]


class RopeShape(ctypes.Structure):
    _fields_ = [("tokens", ctypes.c_int), ("seq_len", ctypes.c_int), ("heads", ctypes.c_int),
                ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int), ("rot_dim", ctypes.c_int),
                ("interleaved", ctypes.c_int), ("max_pos", ctypes.c_int),
                ("q_row_stride", ctypes.c_longlong), ("k_row_stride", ctypes.c_longlong),
                ("v_row_stride", ctypes.c_longlong), ("q_out_row_stride", ctypes.c_longlong),
                ("k_out_row_stride", ctypes.c_longlong)]


class PrefixShape(ctypes.Structure):
    _fields_ = [("n_seq", ctypes.c_int), ("n_groups", ctypes.c_int), ("heads", ctypes.c_int),
                ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int), ("dtype", ctypes.c_int),
                ("page_size", ctypes.c_int), ("max_prefix_pages", ctypes.c_int), ("max_pages", ctypes.c_int),
                ("max_prefix_len", ctypes.c_int), ("max_len", ctypes.c_int),
                ("q_row_stride", ctypes.c_longlong), ("out_row_stride", ctypes.c_longlong),
                ("scale", ctypes.c_float)]


class Split(ctypes.Structure):
    _fields_ = [("batch0", ctypes.c_int), ("batch", ctypes.c_int), ("head0", ctypes.c_int),
                ("heads", ctypes.c_int), ("nb", ctypes.c_int), ("nh", ctypes.c_int)]


P = ctypes.c_void_p
I = ctypes.c_int
LL = ctypes.c_longlong
SZ = ctypes.c_size_t

# name -> (restype, argtypes); every symbol of include/attn_b200.h
SIGNATURES = {
    "attn_last_error": (ctypes.c_char_p, []),
    "attn_device_error": (I, [I, ctypes.POINTER(I)]),
    "attn_version": (I, []),
    "attn_fwd": (None, [P, P, P, P, P]),
    "attn_bwd": (None, [P, P, P, P, P, P, P, P, P]),
    "attn_set_macro_shape": (I, [I, I, I, I]),
    "attn_set_probs_mode": (I, [I]),
    "attn_fwd_ex": (I, [ctypes.POINTER(Shape), I, P, P, P, P, P, P]),
    "attn_bwd_workspace_bytes": (SZ, [ctypes.POINTER(Shape), I]),
    "attn_bwd_ex": (I, [ctypes.POINTER(Shape), I, P, P, P, P, P, P, P, P, P, I, P, SZ, P]),
    "attn_bwd_tc_workspace_bytes": (SZ, [ctypes.POINTER(Shape)]),
    "attn_qkv_workspace_bytes": (SZ, [ctypes.POINTER(QKVShape)]),
    "attn_qkv_proj_ex": (I, [ctypes.POINTER(QKVShape), P, P, P, P, P, P, P, P, P, P, P, SZ, P]),
    "attn_qkv_proj": (None, [P, P, P, P, P, P, P, P, P, P, I, I, I]),
    "attn_decode_workspace_bytes": (SZ, [ctypes.POINTER(DecodeShape)]),
    "attn_decode_ex": (I, [ctypes.POINTER(DecodeShape), P, P, P, P, P, P, P, P, SZ, P]),
    "attn_decode_ptrs_ex": (I, [ctypes.POINTER(DecodeShape), P, P, P, P, P, P, P, P, SZ, P]),
    "attn_decode_static_ex": (I, [ctypes.POINTER(DecodeShape), P, P, P, P, P, P, P, P]),
    "attn_cached_attention": (I, [P, P, P, P, I, I, I, LL, P]),
    "attn_kv_quantize_int8": (I, [P, LL, I, I, LL, P, P, P]),
    "attn_kv_cache_alloc": (I, [ctypes.POINTER(KVCache), I, I, I, I, I]),
    "attn_kv_cache_free": (I, [ctypes.POINTER(KVCache)]),
    "attn_kv_cache_append": (I, [ctypes.POINTER(KVCache), I, I, P, P, P]),
    "attn_page_plan_ex": (I, [ctypes.POINTER(PageShape), P, P, P, P, P, P, P, P, P, P, P, P, P]),
    "attn_rope_table_ex": (I, [ctypes.POINTER(RopeConfig), P, P]),
    "attn_rope_ex": (I, [ctypes.POINTER(RopeShape), I, P, P, P, P, P, P, I, P]),
    "attn_rope_append_ex": (I, [ctypes.POINTER(RopeShape), ctypes.POINTER(PagedKV), I, P, P, P, P, P, P, P, P]),
    "attn_prefix_decode_workspace_bytes": (SZ, [ctypes.POINTER(PrefixShape), ctypes.POINTER(PagedKV)]),
    "attn_prefix_decode_ex": (I, [ctypes.POINTER(PrefixShape), ctypes.POINTER(PagedKV), P, P, P, P, P, P, P, P, P, SZ, P]),
    "attn_shard_range": (I, [LL, I, I, ctypes.POINTER(LL), ctypes.POINTER(LL)]),
    "attn_shard_lpt": (I, [P, I, I, I, P, P]),
    "attn_gather_permute": (I, [P, P, I, I, I, I, I, I, P]),
    "attn_debug_decode_timeout": (I, [I, LL]),
    "attn_debug_qkv_timeout": (I, [I, LL]),
    "attn_cached_attention_host": (None, [P, P, P, P, P, I]),
    "attn_set_decode_macro_shape": (I, [I, I, I]),
    "attn_cached_attention_host_ex": (I, [P, P, P, P, I, I, I, LL, I]),
    "attn_host_cache_release": (I, [P, P]),
    "attn_init": (I, [I]),
    "attn_get_unique_id": (I, [P]),
    "attn_init_rank": (I, [I, I, I, P]),
    "attn_finalize": (I, []),
    "attn_group_size": (I, []),
    "attn_group_sync": (I, [P, I, I]),
    "attn_split_plan": (I, [I, I, I, I, ctypes.POINTER(Split)]),
    "attn_gather_workspace_bytes": (SZ, [ctypes.POINTER(Shape), I, I]),
    "attn_gather_split": (I, [ctypes.POINTER(Shape), I, P, P, P, SZ, P]),
    "attn_gather_rows_workspace_bytes": (SZ, [I, SZ, I]),
    "attn_gather_rows": (I, [P, I, SZ, P, I, P, P, SZ, P]),
    "attn_fwd_multi": (I, [ctypes.POINTER(Shape), I, P, P, P, P, P, I, P, P, P]),
    "attn_decode_multi": (I, [ctypes.POINTER(DecodeShape), P, P, P, P, P, P, P, I, I, P, I, P, P, P, P]),
}
for _name, (_res, _args) in SIGNATURES.items():
    _f = getattr(lib, _name)
    _f.restype = _res
    _f.argtypes = _args


def last_error() -> str:
    return lib.attn_last_error().decode()


def check(status: int):
    if status != OK:
        raise AttnError(status, last_error())


# ---------------------------------------------------------------------------
# raw-pointer API
# ---------------------------------------------------------------------------
def fwd_ex(shape: Shape, dtype, q, k, v, o, lse, stream=0):
    check(lib.attn_fwd_ex(ctypes.byref(shape), dtype, q, k, v, o, lse, stream))


def bwd_workspace_bytes(shape: Shape, dtype) -> int:
    return lib.attn_bwd_workspace_bytes(ctypes.byref(shape), dtype)


def bwd_ex(shape: Shape, dtype, do, q, k, v, o, lse, dq, dk, dv, accumulate, ws, ws_bytes, stream=0):
    check(lib.attn_bwd_ex(ctypes.byref(shape), dtype, do, q, k, v, o, lse, dq, dk, dv,
                          int(accumulate), ws, ws_bytes, stream))


def decode_workspace_bytes(shape: DecodeShape) -> int:
    return lib.attn_decode_workspace_bytes(ctypes.byref(shape))


def decode_ex(shape: DecodeShape, q, kc, vc, ks, vs, lens, out, ws=None, ws_bytes=0, stream=0):
    check(lib.attn_decode_ex(ctypes.byref(shape), q, kc, vc, ks, vs, lens, out, ws, ws_bytes, stream))


def shard_range(n_units: int, world: int, rank: int):
    b, e = LL(), LL()
    check(lib.attn_shard_range(n_units, world, rank, ctypes.byref(b), ctypes.byref(e)))
    return b.value, e.value


def split_plan(batch: int, heads: int, nranks: int, rank: int) -> Split:
    sp = Split()
    check(lib.attn_split_plan(batch, heads, nranks, rank, ctypes.byref(sp)))
    return sp


def shard_lpt(lens, heads: int, world: int):
    """LPT assignment of (seq, head) units; returns (rank per unit, load per rank)."""
    import numpy as np
    lens = np.ascontiguousarray(lens, dtype=np.int32)
    ranks = np.empty(len(lens) * heads, dtype=np.int32)
    load = np.empty(world, dtype=np.int64)
    check(lib.attn_shard_lpt(lens.ctypes.data, len(lens), heads, world, ranks.ctypes.data, load.ctypes.data))
    return ranks, load


# ---------------------------------------------------------------------------
# torch-tensor helpers (device memory + stream plumbing only)
# ---------------------------------------------------------------------------
def _dtype_code(t):
    import torch
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"unsupported dtype {t.dtype}")


def _device() -> int:
    """Number of torch's current device."""
    import torch
    return torch._C._cuda_getDevice()


def _stream():
    """Handle of torch's current stream on the current device."""
    import torch
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def forward_t(q, k, v, heads: int, batch: int, out=None, lse=None, want_lse=True):
    """q,k,v: (batch*T, heads*d) CUDA tensors (fp32 or bf16), row-major."""
    import torch
    rows, width = q.shape
    T = rows // batch
    d = width // heads
    out = torch.empty_like(q) if out is None else out
    if want_lse and lse is None:
        lse = torch.empty(batch * heads * T, dtype=torch.float32, device=q.device)
    shape = Shape(batch, heads, T, d, q.stride(0), out.stride(0))
    fwd_ex(shape, _dtype_code(q), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
           lse.data_ptr() if lse is not None else None, _stream())
    return out, lse


def backward_t(do, q, k, v, o, lse, heads: int, batch: int, dq=None, dk=None, dv=None, accumulate=False):
    import torch
    rows, width = q.shape
    T = rows // batch
    d = width // heads
    shape = Shape(batch, heads, T, d, q.stride(0), o.stride(0))
    dq = torch.zeros_like(q) if dq is None else dq
    dk = torch.zeros_like(q) if dk is None else dk
    dv = torch.zeros_like(q) if dv is None else dv
    nbytes = bwd_workspace_bytes(shape, _dtype_code(q))
    ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
    bwd_ex(shape, _dtype_code(q), do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
           lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), accumulate, ws.data_ptr(), nbytes,
           _stream())
    return dq, dk, dv


def qkv_proj_t(x, wq, wk, wv, bq=None, bk=None, bv=None, fused=False, out=None, workspace=None):
    """Q, K, V = x @ W + b for the three weights in one launch (train_kaggle.cu:152-154).
    x: (M, Kd) fp32 CUDA tensor (any row stride that is a multiple of 4); W: (Kd, N).
    fused=True writes one (M, 3N) tensor whose column blocks are Q, K and V and
    returns (qkv, q_view, k_view, v_view); otherwise returns three (M, N) tensors."""
    import torch
    M, Kd = x.shape
    N = wq.shape[1]
    if fused:
        qkv = torch.empty((M, 3 * N), dtype=torch.float32, device=x.device) if out is None else out
        outs = (qkv[:, :N], qkv[:, N:2 * N], qkv[:, 2 * N:])
    else:
        outs = tuple(torch.empty((M, N), dtype=torch.float32, device=x.device) for _ in range(3)) \
            if out is None else out
    shape = QKVShape(M, Kd, N, x.stride(0), outs[0].stride(0))

    def ptr(t):
        return t.data_ptr() if t is not None else None
    ws_ptr, ws_bytes = (None, 0)
    if workspace is not None:
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    check(lib.attn_qkv_proj_ex(ctypes.byref(shape), x.data_ptr(), wq.data_ptr(), wk.data_ptr(), wv.data_ptr(),
                               ptr(bq), ptr(bk), ptr(bv), outs[0].data_ptr(), outs[1].data_ptr(),
                               outs[2].data_ptr(), ws_ptr, ws_bytes, _stream()))
    return (qkv,) + outs if fused else outs


def decode_t(q, kcache, vcache, lens, heads: int, cap: int, max_len: int, kscale=None, vscale=None,
             out=None, workspace=None):
    """q: (n_seq, H*d) fp32; caches: (n_seq*cap, row_stride) fp32 or int8."""
    import torch
    n_seq, width = q.shape
    d = width // heads
    kv = I8 if kcache.dtype == torch.int8 else F32
    shape = DecodeShape(n_seq, heads, d, kv, kcache.stride(0), cap, max_len)
    out = torch.empty_like(q) if out is None else out
    ws_ptr, ws_bytes = (None, 0)
    if workspace is not None:
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    decode_ex(shape, q.data_ptr(), kcache.data_ptr(), vcache.data_ptr(),
              kscale.data_ptr() if kscale is not None else None,
              vscale.data_ptr() if vscale is not None else None,
              lens.data_ptr() if lens is not None else None, out.data_ptr(), ws_ptr, ws_bytes, _stream())
    return out


def quantize_int8_t(x, heads: int):
    """x: (rows, H*d) fp32 CUDA tensor -> (codes int8 same layout, scales (rows, H) fp32)."""
    import torch
    rows, width = x.shape
    d = width // heads
    codes = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty((rows, heads), dtype=torch.float32, device=x.device)
    check(lib.attn_kv_quantize_int8(x.data_ptr(), rows, heads, d, x.stride(0), codes.data_ptr(),
                                    scales.data_ptr(), _stream()))
    return codes, scales


def gather_permute_t(staging, world, batch, seq_len, heads, head_dim):
    import torch
    out = torch.empty((batch * seq_len, heads * head_dim), dtype=staging.dtype, device=staging.device)
    check(lib.attn_gather_permute(staging.data_ptr(), out.data_ptr(), world, batch, seq_len, heads, head_dim,
                                  _dtype_code(staging), _stream()))
    return out


# ---------------------------------------------------------------------------
# serving over a paged cache
# ---------------------------------------------------------------------------
class PageCache(PagedKV):
    """A paged cache over k and v tensors of (rows, kv_heads * d), which it keeps alive.  An int8 cache brings its
    (rows, kv_heads) fp32 scales."""

    @classmethod
    def of(cls, k, v, kscale=None, vscale=None):
        import torch
        kv = I8 if k.dtype == torch.int8 else _dtype_code(k)
        if v.dtype != k.dtype or v.shape != k.shape or v.stride() != k.stride() or k.dim() != 2 or k.stride(1) != 1:
            raise ValueError("k and v must have one type, shape and layout, with dense rows")
        if not k.is_cuda or v.device != k.device:
            raise ValueError("k and v must be CUDA tensors of one device")
        if kv == I8:
            for x in (kscale, vscale):
                if x is None or x.dim() != 2 or x.shape != (k.shape[0], kscale.shape[1]) or not x.is_contiguous():
                    raise ValueError("an int8 cache needs dense kscale and vscale of (rows, kv_heads)")
                if x.dtype != torch.float32 or x.device != k.device:
                    raise TypeError("kscale and vscale must be fp32 tensors of the cache's device")
        c = cls(kv, k.shape[0], k.stride(0), k.data_ptr(), v.data_ptr(), _ptr(kscale), _ptr(vscale))
        c.tensors = (k, v, kscale, vscale)
        c.device, c.width, c.scale_heads = k.get_device(), k.shape[1], kscale.shape[1] if kv == I8 else None
        return c


def _ptr(t):
    return t.data_ptr() if t is not None else None


# The shapes of these calls stand beside their tensors, so each tensor is looked at: what the library reads and writes
# by a shape has to lie within it, on the current device.  (In one pass over few attributes: it counts in calls of a
# few microseconds.)
def _dense(device, *given):
    """(name, tensor, dtype, elements): the tensor (None: not given) is a dense one of so many elements or more."""
    for name, t, dtype, n in given:
        if t is not None and (t.dtype is not dtype or not t.is_contiguous() or t.numel() < n or t.get_device() != device):
            if t.dtype is not dtype:
                raise TypeError(f"{name} is {t.dtype}, not {dtype}")
            raise ValueError(f"{name}, {tuple(t.shape)} of strides {t.stride()} on {t.device}, is not {n} dense elements on device {device}")


def _rows(device, dtype, name, t, rows, width, stride):
    """t (None: not given) is a tensor of dtype with `rows` rows of `width` elements, `stride` apart (0: width), as
    (rows, width) or, where it is dense, in any shape whose last dimension lies within a row."""
    if t is None:
        return
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, not {dtype}")
    stride, shape, steps = stride or width, t.shape, t.stride()
    fits = len(shape) == 2 and shape[0] >= rows and shape[1] >= width and steps[1] == 1 and (steps[0] == stride or rows == 1) or \
        rows <= 0 or width <= 0 or \
        stride == width and t.is_contiguous() and t.numel() >= rows * width and shape[-1] <= width
    if not fits or t.get_device() != device:
        raise ValueError(f"{name}, {tuple(shape)} of strides {steps} on {t.device}, is not {rows} rows of {width}, {stride} apart, "
                         f"on device {device}")


def _cache_holds(device, cache, kv_heads, head_dim):
    """The tensors of a PageCache hold rows of these heads (a PagedKV of bare addresses cannot be looked at)."""
    if isinstance(cache, PageCache):
        if cache.device != device:
            raise ValueError(f"the cache is on device {cache.device}, not {device}")
        if cache.width < kv_heads * head_dim:
            raise ValueError(f"cache rows of {cache.width} elements hold no {kv_heads} heads of {head_dim}")
        if cache.scale_heads not in (None, kv_heads):
            raise ValueError(f"cache scales of {cache.scale_heads} heads, not {kv_heads}")


def page_outputs(shape: PageShape, device="cuda"):
    """Tensors that page_plan_t writes for this shape, by name."""
    import torch
    out = {k: torch.empty(n, dtype=torch.int32, device=device)
           for k, n in (("lens", shape.n_seq), ("cu_new", shape.n_seq + 1), ("positions", shape.max_tokens),
                        ("token_seq", shape.max_tokens), ("counts", 4))}
    out["slot_map"] = torch.empty(shape.max_tokens, dtype=torch.int64, device=device)
    return out


def page_plan_t(shape: PageShape, lens, new_lens, free_pages, free_count, block_table, out, pos_base=None):
    """attn_page_plan_ex: int32 CUDA tensors; `out` as page_outputs makes it (slot_map int64).  Writes `out`, the new
    entries of block_table and the returned pages in free_pages; out["lens"] and out["counts"][:1] are the next step's
    lens and free_count."""
    import torch
    on, n, rows, i32 = _device(), shape.n_seq, shape.max_tokens, torch.int32
    _dense(on, ("lens", lens, i32, n), ("new_lens", new_lens, i32, n), ("pos_base", pos_base, i32, n), ("free_pages", free_pages, i32, shape.n_pages),
           ("free_count", free_count, i32, 1), ("out['lens']", out["lens"], i32, n), ("out['cu_new']", out["cu_new"], i32, n + 1),
           ("out['slot_map']", out["slot_map"], torch.int64, rows), ("out['positions']", out["positions"], i32, rows),
           ("out['token_seq']", out.get("token_seq"), i32, rows), ("out['counts']", out["counts"], i32, 4))
    _rows(on, i32, "block_table", block_table, n, shape.max_pages, shape.table_stride)
    check(lib.attn_page_plan_ex(shape, lens.data_ptr(), new_lens.data_ptr(), _ptr(pos_base), free_pages.data_ptr(),
                                free_count.data_ptr(), block_table.data_ptr(), out["lens"].data_ptr(),
                                out["cu_new"].data_ptr(), out["slot_map"].data_ptr(), out["positions"].data_ptr(),
                                _ptr(out.get("token_seq")), out["counts"].data_ptr(), _stream()))
    return out


def rope_table_t(config: RopeConfig, device="cuda"):
    """The (max_pos, rot_dim / 2, 2) fp32 table of cosines and sines of a configuration."""
    import torch
    table = torch.empty((config.max_pos, config.rot_dim // 2, 2), dtype=torch.float32, device=device)
    check(lib.attn_rope_table_ex(config, table.data_ptr(), _stream()))
    return table


def rope_t(shape: RopeShape, table, positions, q, k, q_out, k_out, transpose=False):
    """attn_rope_ex on (tokens, heads * d) fp32 or bf16 tensors; positions int32 or None; k and k_out may be None."""
    import torch
    on, n, d, dtype = _device(), shape.tokens, shape.head_dim, q.dtype
    _dense(on, ("table", table, torch.float32, shape.max_pos * shape.rot_dim), ("positions", positions, torch.int32, n))
    _rows(on, dtype, "q", q, n, shape.heads * d, shape.q_row_stride)
    _rows(on, dtype, "k", k, n, shape.kv_heads * d, shape.k_row_stride)
    _rows(on, dtype, "q_out", q_out, n, shape.heads * d, shape.q_out_row_stride)
    _rows(on, dtype, "k_out", k_out, n, shape.kv_heads * d, shape.k_out_row_stride)
    check(lib.attn_rope_ex(shape, _dtype_code(q), _ptr(table), _ptr(positions), q.data_ptr(), _ptr(k),
                           q_out.data_ptr(), _ptr(k_out), int(transpose), _stream()))
    return q_out, k_out


def rope_append_t(shape: RopeShape, cache: PagedKV, table, positions, slot_map, q, k, v, q_out):
    """attn_rope_append_ex: positions int32 or None, slot_map int64."""
    import torch
    on, n, d, heads, dtype = _device(), shape.tokens, shape.head_dim, shape.kv_heads, q.dtype
    _dense(on, ("table", table, torch.float32, shape.max_pos * shape.rot_dim), ("positions", positions, torch.int32, n),
           ("slot_map", slot_map, torch.int64, n))
    _rows(on, dtype, "q", q, n, shape.heads * d, shape.q_row_stride)
    _rows(on, dtype, "k", k, n, heads * d, shape.k_row_stride)
    _rows(on, dtype, "v", v, n, heads * d, shape.v_row_stride)
    _rows(on, dtype, "q_out", q_out, n, shape.heads * d, shape.q_out_row_stride)
    _cache_holds(on, cache, heads, d)
    check(lib.attn_rope_append_ex(shape, cache, _dtype_code(q), _ptr(table), _ptr(positions), slot_map.data_ptr(),
                                  q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), _stream()))
    return q_out


def prefix_decode_workspace_bytes(shape: PrefixShape, cache: PagedKV) -> int:
    return lib.attn_prefix_decode_workspace_bytes(shape, cache)


def prefix_decode_t(shape: PrefixShape, cache: PagedKV, q, group_begin, prefix_table, prefix_lens, block_table, lens,
                    out, lse=None, workspace=None):
    """attn_prefix_decode_ex: q and out (n_seq, heads * d); tables and lengths int32; group_begin, prefix_table and
    prefix_lens may be None when shape.n_groups is 0."""
    import torch
    on, n, groups, heads, d, i32 = _device(), shape.n_seq, shape.n_groups, shape.heads, shape.head_dim, torch.int32
    dtype = torch.bfloat16 if shape.dtype == BF16 else torch.float32
    _dense(on, ("lens", lens, i32, n), ("lse", lse, torch.float32, n * heads),
           ("workspace", workspace, workspace.dtype if workspace is not None else None, 0))
    if groups > 0:
        _dense(on, ("group_begin", group_begin, i32, groups + 1), ("prefix_lens", prefix_lens, i32, groups))
        _rows(on, i32, "prefix_table", prefix_table, groups, shape.max_prefix_pages, 0)
    _rows(on, i32, "block_table", block_table, n, shape.max_pages, 0)
    _rows(on, dtype, "q", q, n, heads * d, shape.q_row_stride)
    _rows(on, dtype, "out", out, n, heads * d, shape.out_row_stride)
    _cache_holds(on, cache, shape.kv_heads, d)
    check(lib.attn_prefix_decode_ex(shape, cache, q.data_ptr(), _ptr(group_begin), _ptr(prefix_table),
                                    _ptr(prefix_lens), block_table.data_ptr(), lens.data_ptr(), out.data_ptr(),
                                    _ptr(lse), _ptr(workspace),
                                    workspace.numel() * workspace.element_size() if workspace is not None else 0,
                                    _stream()))
    return out

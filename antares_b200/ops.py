"""torch-tensor front ends of the C ABI.  Tensors must live on a CUDA device; launches go to
torch's current stream (the reference launches on the NULL stream, frameworks/pytorch/main_ops.cc:44).
Nothing here computes on the CPU: a CPU tensor is an error, not a fallback.
"""
import torch

from . import _lib
from ._lib import F16, F32, call, fast

_DT = {torch.float16: F16, torch.float32: F32}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _chk(t, name, dtype=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("%s must be a CUDA tensor (antares_b200 has no CPU path)" % name)
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    if dtype is not None and t.dtype != dtype:
        raise ValueError("%s must be %s, got %s" % (name, dtype, t.dtype))
    return t.data_ptr()


def _code(dtype):
    try:
        return _DT[dtype]
    except KeyError:
        raise ValueError("dtype %s is outside the built kernel family (float16, float32)" % dtype)


def device_info(device=0):
    import ctypes
    buf = (ctypes.c_int * 8)()
    call("ab200_device_info", int(device), ctypes.cast(buf, ctypes.c_void_p))
    keys = ["sm_count", "smem_optin_bytes", "l2_bytes", "sm_clock_khz", "mem_clock_khz", "bus_width_bits", "cc", "max_threads"]
    return dict(zip(keys, list(buf)))


def w4_unpack(qweight):
    Kp, N = qweight.shape
    out = torch.empty((Kp * 8, N), dtype=torch.uint8, device=qweight.device)
    call("ab200_w4_unpack", _chk(qweight, "qweight", torch.int32), Kp * 8, N, out.data_ptr(), _stream())
    return out


def w4_pack(q):
    K, N = q.shape
    out = torch.empty((K // 8, N), dtype=torch.int32, device=q.device)
    call("ab200_w4_pack", _chk(q, "q", torch.uint8), K, N, out.data_ptr(), _stream())
    return out


def w4_dequant(qweight, scales, group=128):
    Kp, N = qweight.shape
    out = torch.empty((Kp * 8, N), dtype=scales.dtype, device=qweight.device)
    call("ab200_w4_dequant", _chk(qweight, "qweight", torch.int32), _chk(scales, "scales"), Kp * 8, N, group,
         _code(scales.dtype), out.data_ptr(), _stream())
    return out


def _gemm_shapes(x, qweight, scales, group):
    Kp, N = qweight.shape
    K = Kp * 8
    if x.shape[-1] != K:
        raise ValueError("x has %d features but qweight packs %d" % (x.shape[-1], K))
    M = x.numel() // K
    if group is None:
        group = K // scales.shape[0]
    if scales.shape != (K // group, N):
        raise ValueError("scales shape %s does not match [K/group=%d, N=%d]" % (tuple(scales.shape), K // group, N))
    if scales.dtype != x.dtype:
        raise ValueError("x (%s) and scales (%s) must share a dtype" % (x.dtype, scales.dtype))
    return M, K, N, group


def w4a16_gemv(x, qweight, scales, out=None, group=None):
    """out[..., N] = x[..., K] . dequant(qweight, scales); M = x.numel()/K <= 16."""
    if out is None and group is None:
        y = fast().w4a16(1, x, qweight, scales)
        if y is not None:
            return y
    M, K, N, group = _gemm_shapes(x, qweight, scales, group)
    if out is None:
        out = torch.empty(tuple(x.shape[:-1]) + (N,), dtype=x.dtype, device=x.device)
    elif out.numel() != M * N or out.dtype != x.dtype:
        raise ValueError("out must hold %d elements of %s" % (M * N, x.dtype))
    call("ab200_w4a16_gemv", _chk(x, "x"), _chk(qweight, "qweight", torch.int32), _chk(scales, "scales"),
         _chk(out, "out"), M, K, N, group, _code(x.dtype), _stream())
    return out


def w4a16_gemv_residual(x, qweight, scales, resid, group=None):
    """resid_f32[..., N] += fp16_round(x . W)."""
    M, K, N, group = _gemm_shapes(x, qweight, scales, group)
    if resid.numel() != M * N:
        raise ValueError("resid must hold %d elements" % (M * N))
    call("ab200_w4a16_gemv_residual", _chk(x, "x", torch.float16), _chk(qweight, "qweight", torch.int32),
         _chk(scales, "scales", torch.float16), _chk(resid, "resid", torch.float32), M, K, N, group, _stream())
    return resid


def w4a16_gemm(x, qweight, scales, out=None, group=None):
    """Prefill contraction on tensor cores."""
    if out is None and group is None:
        y = fast().w4a16(2, x, qweight, scales)
        if y is not None:
            return y
    Kp, N = qweight.shape
    K = Kp * 8
    M = x.numel() // K
    if group is None:
        group = K // scales.shape[0]
    if out is None:
        out = torch.empty(tuple(x.shape[:-1]) + (N,), dtype=x.dtype, device=x.device)
    call("ab200_w4a16_gemm", _chk(x, "x"), _chk(qweight, "qweight", torch.int32), _chk(scales, "scales"),
         _chk(out, "out"), M, K, N, group, _code(x.dtype), _stream())
    return out


def w4a16_matmul(x, qweight, scales, out=None, group=None):
    """The exported op of samples/05_llama2_7b_int4.py:135-144 for any batch: decode kernel up to
    16 rows, tensor-core kernel above."""
    if out is None and group is None:
        y = fast().w4a16(0, x, qweight, scales)
        if y is not None:
            return y
    M = x.numel() // (qweight.shape[0] * 8)
    if M <= 16:
        return w4a16_gemv(x, qweight, scales, out, group)
    return w4a16_gemm(x, qweight, scales, out, group)


def sigmoid(x, out=None):
    if out is None:
        y = fast().sigmoid(x)
        if y is not None:
            return y
        out = torch.empty_like(x)
    call("ab200_sigmoid", _chk(x, "x"), _chk(out, "out", x.dtype), x.numel(), _code(x.dtype), _stream())
    return out


def rmsnorm_vsum(x, vsum, weight, inv_n, eps=1e-6, out=None):
    if out is None:
        out = torch.empty_like(x)
    call("ab200_rmsnorm_vsum", _chk(x, "x"), _chk(vsum, "vsum", torch.float32), _chk(weight, "weight", x.dtype),
         _chk(out, "out", x.dtype), x.numel(), float(inv_n), float(eps), _code(x.dtype), _stream())
    return out


def rmsnorm(x, weight, eps=1e-6, out=None):
    if out is None:
        y = fast().rmsnorm(x, weight, eps)
        if y is not None:
            return y
    cols = x.shape[-1]
    rows = x.numel() // cols
    if out is None:
        out = torch.empty(x.shape, dtype=torch.float16, device=x.device)
    call("ab200_rmsnorm", _chk(x, "x"), _code(x.dtype), _chk(weight, "weight", torch.float16),
         _chk(out, "out", torch.float16), rows, cols, float(eps), _stream())
    return out


def rope(x, pos, inv_freq, out=None):
    if out is None:
        y = fast().rope(x, pos, inv_freq)
        if y is not None:
            return y
    rows, H, D = x.shape
    if out is None:
        out = torch.empty_like(x)
    call("ab200_rope", _chk(x, "x"), _chk(inv_freq, "inv_freq", torch.float32),
         _chk(pos, "pos", torch.int32), _chk(out, "out", x.dtype), rows, H, D, _code(x.dtype), _stream())
    return out


def softmax(x, out=None):
    if out is None:
        y = fast().softmax(x)
        if y is not None:
            return y
    cols = x.shape[-1]
    rows = x.numel() // cols
    if out is None:
        out = torch.empty_like(x)
    call("ab200_softmax", _chk(x, "x"), _chk(out, "out", x.dtype), rows, cols, _code(x.dtype), _stream())
    return out


def attention_decode(q, k_cache, v_cache, seq_len_dev, scale, out=None, kv_stride=None, max_seq=None, seq_len_add=0):
    H, D = q.shape
    if kv_stride is None:
        kv_stride = k_cache.stride(0)
    if max_seq is None:
        max_seq = k_cache.shape[0]
    if out is None:
        out = torch.empty_like(q)
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError("q, k_cache and v_cache must share a dtype")
    call("ab200_attention_decode", _chk(q, "q"), k_cache.data_ptr(), v_cache.data_ptr(),
         _chk(out, "out", q.dtype), _chk(seq_len_dev, "seq_len_dev", torch.int32), int(seq_len_add), int(max_seq), H, D,
         int(kv_stride), float(scale), _code(q.dtype), _stream())
    return out


def set_option(name, value):
    """Process-wide tuning knob (gemv_cluster, gemv_impl)."""
    call("ab200_set_option", name.encode(), int(value))


def kernel_status():
    """Reads and clears the device status word; raises Ab200Error(ETIMEOUT) if a bounded wait ran out."""
    import ctypes
    v = ctypes.c_int(0)
    call("ab200_kernel_status", ctypes.cast(ctypes.pointer(v), ctypes.c_void_p))
    return v.value


PRO_PLAIN, PRO_RMSNORM, PRO_SILU_MUL = 0, 1, 2
EPI_F16, EPI_RESIDUAL, EPI_F32 = 0, 1, 2


def gemv_workspace_bytes(M, K, N):
    return int(_lib.load().ab200_w4a16_gemv_workspace_bytes(int(M), int(K), int(N)))


def w4a16_gemv_fused(x, qweight, scales, out, prologue=PRO_PLAIN, epilogue=EPI_F16, norm_weight=None, eps=1e-6,
                     group=None, workspace=None):
    """One-launch decode projection: optional RMSNorm / SiLU*up on the way in, optional residual
    add on the way out.  x: fp16 [M,K] (plain), fp32 [M,K] (RMSNorm) or fp16 [M,2K] (SiLU*up)."""
    Kp, N = qweight.shape
    K = Kp * 8
    xk = 2 * K if prologue == PRO_SILU_MUL else K
    M = x.numel() // xk
    if group is None:
        group = K // scales.shape[0]
    want_x = torch.float32 if prologue == PRO_RMSNORM else torch.float16
    want_o = torch.float16 if epilogue == EPI_F16 else torch.float32
    if out.numel() != M * N:
        raise ValueError("out must hold %d elements" % (M * N))
    ws_ptr, ws_bytes = (0, 0) if workspace is None else (_chk(workspace, "workspace"), workspace.numel() * workspace.element_size())
    call("ab200_w4a16_gemv_fused", _chk(x, "x", want_x), int(prologue),
         0 if norm_weight is None else _chk(norm_weight, "norm_weight", torch.float16), float(eps),
         _chk(qweight, "qweight", torch.int32), _chk(scales, "scales", torch.float16), _chk(out, "out", want_o), int(epilogue),
         M, K, N, group, ws_ptr, ws_bytes, _stream())
    return out


def w4a16_gemv_tiled(x, qweight_tiled, scales_tiled, out, prologue=PRO_PLAIN, epilogue=EPI_F16, norm_weight=None, eps=1e-6, group=128):
    """w4a16_gemv_fused on tile-major weights (packing.tile_weights): qweight_tiled [N/128, K/8, 128]."""
    K, N = qweight_tiled.shape[1] * 8, qweight_tiled.shape[0] * qweight_tiled.shape[2]
    xk = x.shape[-1] // 2 if prologue == PRO_SILU_MUL else x.shape[-1]
    if xk != K:
        raise ValueError("x has %d values per row, the weights %d rows" % (xk, K))
    M = x.numel() // x.shape[-1]
    call("ab200_w4a16_gemv_tiled", _chk(x, "x"), prologue, 0 if norm_weight is None else _chk(norm_weight, "norm_weight", torch.float16), float(eps),
         _chk(qweight_tiled, "qweight_tiled", torch.int32), _chk(scales_tiled, "scales_tiled", torch.float16), _chk(out, "out"),
         epilogue, M, K, N, group, _stream())
    return out


def eltwise_program(prog, consts, inputs, out=None, out_dtype=None):
    """Runs a stack program (ir.compile_elementwise) over same-sized fp16/fp32 tensors."""
    import ctypes
    n = inputs[0].numel()
    for t in inputs:
        if t.numel() != n:
            raise ValueError("element-wise inputs must all hold %d elements" % n)
    if out is None:
        out = torch.empty_like(inputs[0], dtype=out_dtype or inputs[0].dtype)
    elif out.numel() != n:
        raise ValueError("out must hold %d elements" % n)
    ops_b = (ctypes.c_ubyte * len(prog))(*[int(o) for o, _ in prog])
    args_b = (ctypes.c_ubyte * len(prog))(*[int(a) for _, a in prog])
    cst = (ctypes.c_float * max(1, len(consts)))(*[float(c) for c in consts])
    ptrs = (ctypes.c_void_p * len(inputs))(*[_chk(t, "input") for t in inputs])
    dts = (ctypes.c_int * len(inputs))(*[_code(t.dtype) for t in inputs])
    call("ab200_eltwise_vm", ctypes.cast(ops_b, ctypes.c_void_p), ctypes.cast(args_b, ctypes.c_void_p), len(prog), ctypes.cast(cst, ctypes.c_void_p),
         len(consts), ctypes.cast(ptrs, ctypes.c_void_p), ctypes.cast(dts, ctypes.c_void_p), len(inputs), _chk(out, "out"), _code(out.dtype), n, _stream())
    return out


def row_program(rp, mats, cols, out=None, out_dtype=None):
    """Runs a compiled reduce + map chain (ir.compile_row_program) over [..., cols] tensors: `mats` the
    full-shape inputs, `cols` the [cols] vectors, in the program's operand order."""
    import ctypes
    shape = mats[0].shape
    ncols = shape[-1]
    rows = mats[0].numel() // ncols
    for t in mats:
        if t.shape != shape:
            raise ValueError("row program: full-shape inputs must share one shape (%s vs %s)" % (tuple(t.shape), tuple(shape)))
    for t in cols:
        if t.numel() != ncols:
            raise ValueError("row program: a column vector must hold %d elements" % ncols)
    if out is None:
        dt = out_dtype or (torch.float32 if any(a.dtype == torch.float32 for a in list(mats) + list(cols)) else torch.float16)
        out = torch.empty(shape, dtype=dt, device=mats[0].device)
    elif out.numel() != mats[0].numel():
        raise ValueError("out must hold %d elements" % mats[0].numel())
    flat = [oa for _, prog in rp["stages"] for oa in prog]
    ops_b = (ctypes.c_ubyte * len(flat))(*[int(o) for o, _ in flat])
    args_b = (ctypes.c_ubyte * len(flat))(*[int(a) for _, a in flat])
    lens = (ctypes.c_int * len(rp["stages"]))(*[len(prog) for _, prog in rp["stages"]])
    kinds = (ctypes.c_int * len(rp["stages"]))(*[int(k) for k, _ in rp["stages"]])
    consts = rp["consts"]
    cst = (ctypes.c_float * max(1, len(consts)))(*[float(c) for c in consts])
    mp = (ctypes.c_void_p * len(mats))(*[_chk(t, "input") for t in mats])
    md = (ctypes.c_int * len(mats))(*[_code(t.dtype) for t in mats])
    cp = (ctypes.c_void_p * max(1, len(cols)))(*[_chk(t, "column vector") for t in cols])
    cd = (ctypes.c_int * max(1, len(cols)))(*[_code(t.dtype) for t in cols])
    P = ctypes.c_void_p
    call("ab200_rowreduce_vm", ctypes.cast(ops_b, P), ctypes.cast(args_b, P), ctypes.cast(lens, P), ctypes.cast(kinds, P), len(rp["stages"]),
         ctypes.cast(cst, P), len(consts), ctypes.cast(mp, P), ctypes.cast(md, P), len(mats), ctypes.cast(cp, P), ctypes.cast(cd, P), len(cols),
         _chk(out, "out"), _code(out.dtype), rows, ncols, _stream())
    return out


# ---- a paged KV cache held in 8 bits ---------------------------------------------------------------------------
# A layer's cache is four tensors (k, v, k_scale, v_scale): int8 [pages, kv heads, page rows, 128] twice, fp32 [pages, kv
# heads, page rows / 16] twice; a value is code * scale.  kv_cache.PagedKV8Cache keeps the pages of many sequences.
# `page_table` int32 [S, max_pages]: position p of sequence s is row p % page_rows of page table[s, p // page_rows].  A table that
# is only read may be one row expanded over the sequences.
# `pos0` int32 [S]: the position of each sequence's first row of the call.  `cu_rows` int32 [S + 1]: which rows are whose
# (None: as many for each).  The tensors' device is the one that works, whichever is current.

def _kv8_args(cache, page_table, pos0, cu_rows, T, q=None, writes=False):
    """The cache and row arguments of a kv8 entry point; checks what only tensors can say."""
    k, v, ks, vs = cache
    if k.dim() != 4 or k.shape[3] != 128 or v.shape != k.shape:
        raise ValueError("a kv8 cache holds k and v int8 [pages, kv heads, page rows, 128], got %s and %s" % (tuple(k.shape), tuple(v.shape)))
    pages, heads, rows, _ = k.shape
    if pages == 0 or heads == 0:
        raise ValueError("a kv8 cache with no heads or no pages holds nothing, got %s" % (tuple(k.shape),))
    if rows < 16 or rows & (rows - 1):
        raise ValueError("a kv8 cache's pages hold a power of two of rows, 16 or more; got %d" % rows)
    if ks.shape != (pages, heads, rows // 16) or vs.shape != ks.shape:
        raise ValueError("a kv8 cache holds scales fp32 %s, got %s and %s" % ((pages, heads, rows // 16), tuple(ks.shape), tuple(vs.shape)))
    if page_table.dim() != 2 or page_table.dtype != torch.int32 or not page_table.is_cuda or (page_table.stride(1) != 1 and page_table.shape[1] > 1):
        raise ValueError("page_table must be a CUDA int32 tensor [sequences, pages] with consecutive columns")
    S = page_table.shape[0]
    stride = page_table.stride(0) if S > 1 else page_table.shape[1]
    if stride < page_table.shape[1] and (writes or stride):
        raise ValueError("the rows of page_table may not overlap%s" % (" where pages are written" if stride == 0 else ""))
    if pos0.numel() != S or (cu_rows is not None and cu_rows.numel() != S + 1):
        raise ValueError("%d sequences need %d positions in pos0 and %d offsets in cu_rows" % (S, S, S + 1))
    for t in (v, ks, vs, page_table, pos0, cu_rows, q):
        if t is not None and t.device != k.device:
            raise ValueError("the tensors of a kv8 call lie on one device (%s and %s)" % (k.device, t.device))
    return (_chk(k, "k cache", torch.int8), _chk(v, "v cache", torch.int8), _chk(ks, "k_scale", torch.float32), _chk(vs, "v_scale", torch.float32),
            pages, rows, heads, page_table.data_ptr(), stride, page_table.shape[1], _chk(pos0, "pos0", torch.int32),
            0 if cu_rows is None else _chk(cu_rows, "cu_rows", torch.int32), S, T)


def _rows3(t, name, dtype, T=None, heads=None):
    """Pointer and row stride of [T, heads, 128] rows; the heads of a row lie together."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("%s must be a CUDA tensor (antares_b200 has no CPU path)" % name)
    if t.dim() != 3 or t.shape[2] != 128 or (T is not None and t.shape[0] != T) or (heads is not None and t.shape[1] != heads):
        raise ValueError("%s must be [%s, %s, 128], got %s" % (name, "rows" if T is None else T, "heads" if heads is None else heads, tuple(t.shape)))
    if t.dtype != dtype:
        raise ValueError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if t.numel() and (t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != 128)):
        raise ValueError("the heads of a row of %s must lie together" % name)
    return t.data_ptr(), t.stride(0) if t.shape[0] > 1 else t.shape[1] * 128


def _disjoint(out, name, *others):
    """A result lies over no input (a cache's pages are read by other rows long after a row's result is stored)."""
    a, b = out.data_ptr(), out.data_ptr() + out.numel() * out.element_size()
    for t in others:
        if t is not None and t.numel() and t.data_ptr() < b and a < t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size():
            raise ValueError("%s may not lie over an input or another result" % name)


def _rows_meet(a, b):
    """Whether two tensors of as many rows, as _rows3 takes them, have a byte in common: rows may lie between one another's, as
    slices of one projection's result do."""
    T, e = a.shape[0], a.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, wa, sa), (b0, wb, sb) = ((t.data_ptr(), t.shape[1] * 128 * t.element_size(), t.stride(0) * t.element_size()) for t in (a, b))
    if T == 1 or a0 + (T - 1) * sa + wa <= b0 or b0 + (T - 1) * sb + wb <= a0:
        return a0 < b0 + (T - 1) * sb + wb and b0 < a0 + (T - 1) * sa + wa
    import numpy as np
    at = np.arange(T, dtype=np.int64) * sa + (a0 - b0)     # a's rows, counted from b's first
    j = np.clip(at // max(sb, e), 0, T - 1)                # the last of b's rows that begins at or before each, and the next
    return any(bool(((at < n * sb + wb) & (n * sb < at + wa)).any()) for n in (j, np.minimum(j + 1, T - 1)))


def kv8_append(cache, k, v, page_table, pos0, cu_rows=None, q=None, inv_freq=None, q_out=None):
    """Writes rows k, v [T, kv heads, 128] into the cache; with inv_freq, k rotated by halves at its positions, and q [T, query
    heads, 128] too: returns the rotated queries (q_out, which may be q but not lie over k, v or other rows of q), else None."""
    if q_out is None:
        y = fast().kv8_append(cache, k, v, page_table, pos0, cu_rows, q, inv_freq)
        if y is not None:
            return None if q is None else y
    T = k.shape[0]
    if q_out is not None and q is None:
        raise ValueError("q_out without q")
    if q is not None and inv_freq is None:
        raise ValueError("q is only rotated: it needs inv_freq")
    args = _kv8_args(cache, page_table, pos0, cu_rows, T, k, writes=True)
    kp, k_stride = _rows3(k, "k", k.dtype, heads=args[6])
    vp, v_stride = _rows3(v, "v", k.dtype, T, args[6])
    fp = 0
    if inv_freq is not None:
        fp = _chk(inv_freq, "inv_freq", torch.float32)
        if inv_freq.numel() < 64:
            raise ValueError("inv_freq must hold 64 values")
    qp = q_stride = qo = qo_stride = hq = zero = 0
    if q is not None:
        qp, q_stride = _rows3(q, "q", k.dtype, T)
        hq = q.shape[1]
        if q_out is None:
            zero, q_out = 1, (torch.empty if args[12] else torch.zeros)(q.shape, dtype=q.dtype, device=q.device)
        qo, qo_stride = _rows3(q_out, "q_out", k.dtype, T, hq)
        for t, name in ((k, "k"), (v, "v"), (q, "q")):
            if _rows_meet(q_out, t) and not (name == "q" and qo == qp and (qo_stride == q_stride or T == 1)):
                raise ValueError("q_out may not lie over %s%s" % (name, " unless it is q" if name == "q" else ""))
    for t in (v, q, q_out, inv_freq):
        if t is not None and t.device != k.device:
            raise ValueError("the tensors of a kv8 call lie on one device")
    with torch.cuda.device(k.device):
        call("ab200_kv8_append", *args, kp, vp, k_stride, v_stride, qp, q_stride, qo, qo_stride, hq, fp, zero, _code(k.dtype), _stream())
    return q_out


def kv8_read(cache, page_table, pos0, rows, cu_rows=None, dtype=torch.float16, out=None):
    """The values held at the rows' positions, (k, v) [rows, kv heads, 128] each; zeros outside the table.  out: a pair of
    tensors to write to, whose rows that are no sequence's stay as they are (new tensors: zeros)."""
    if out is None:
        y = fast().kv8_read(cache, page_table, pos0, rows, cu_rows, _DT.get(dtype, -1))
        if y is not None:
            return y
    args = _kv8_args(cache, page_table, pos0, cu_rows, rows)
    zero = out is None
    if out is None:
        make = torch.empty if args[12] else torch.zeros
        out = tuple(make((rows, args[6], 128), dtype=dtype, device=cache[0].device) for _ in range(2))
    dtype = out[0].dtype
    for t in out:
        _rows3(t, "out", dtype, rows, args[6])
        if not t.is_contiguous() or t.device != cache[0].device:
            raise ValueError("out must be contiguous and on the cache's device")
        _disjoint(t, "out", *cache)
    _disjoint(out[0], "out", out[1])
    with torch.cuda.device(cache[0].device):
        call("ab200_kv8_read", *args, out[0].data_ptr(), out[1].data_ptr(), int(zero), _code(dtype), _stream())
    return out[0], out[1]


def kv8_attention_workspace_bytes(S, T, max_rows, Hq, Hkv):
    return int(_lib.load().ab200_kv8_attention_workspace_bytes(int(S), int(T), int(max_rows), int(Hq), int(Hkv)))


def _kv8_workspace(workspace, S, T, max_rows, Hq, Hkv, device):
    """(pointer, bytes, the tensor that holds them).  Without one of the caller's: memory of this call alone, so that two
    streams or two captured graphs never share it."""
    if workspace is None:
        n = kv8_attention_workspace_bytes(S, T, max_rows, Hq, Hkv)
        if n == 0:
            return 0, 0, None
        workspace = torch.empty(n, dtype=torch.uint8, device=device)
    elif workspace.device != device:
        raise ValueError("workspace must lie on %s" % device)
    return _chk(workspace, "workspace"), workspace.numel() * workspace.element_size(), workspace


def kv8_attention(q, cache, page_table, pos0, cu_rows=None, max_rows=None, scale=None, out=None, workspace=None):
    """Row r of sequence s, q [T, query heads, 128], over the positions 0 .. pos0[s] + r of the cache, which holds them already
    (kv8_append); kv head = query head // (query heads / kv heads).  Rows with no position to attend to are zeros, and so are
    rows that are no sequence's in a new result (in `out` they stay as they are).  max_rows: the most rows of a sequence,
    a hint.  out may be q where q is contiguous."""
    if out is None and workspace is None:
        y = fast().kv8_attention(q, cache, page_table, pos0, cu_rows, max_rows, scale)
        if y is not None:
            return y
    T, hq = q.shape[0], q.shape[1]
    args = _kv8_args(cache, page_table, pos0, cu_rows, T, q)
    qp, q_stride = _rows3(q, "q", q.dtype)
    if hq == 0 or hq % args[6]:
        raise ValueError("%d query heads are not a multiple of %d kv heads" % (hq, args[6]))
    S = args[12]
    if max_rows is None:
        max_rows = T if cu_rows is not None else (T // S if S else 0)
    zero = out is None
    if out is None:
        out = (torch.empty if S else torch.zeros)(q.shape, dtype=q.dtype, device=q.device)
    else:
        if out.shape != q.shape or out.device != q.device:
            raise ValueError("out must be %s on %s" % (tuple(q.shape), q.device))
        _chk(out, "out", q.dtype)
        if not (out.data_ptr() == q.data_ptr() and q.is_contiguous()):
            _disjoint(out, "out", q)
        _disjoint(out, "out", *cache)
    scale = 128 ** -0.5 if scale is None else scale
    with torch.cuda.device(q.device):
        ws, ws_bytes, held = _kv8_workspace(workspace, S, T, max_rows, hq, args[6], q.device)
        call("ab200_kv8_attention", qp, q_stride, out.data_ptr(), *args, int(max_rows), hq, 128, float(scale), int(zero), _code(q.dtype), ws, ws_bytes, _stream())
    return out


def kv8_step(q, k, v, cache, page_table, pos0, inv_freq=None, scale=None, out=None, workspace=None):
    """A decode step's kv8_append and kv8_attention in one call: q [T, query heads, 128], k, v [T, kv heads, 128], T / S rows of
    each sequence, rotated if inv_freq is given."""
    if out is None and workspace is None:
        y = fast().kv8_step(q, k, v, cache, page_table, pos0, inv_freq, scale)
        if y is not None:
            return y
    T, hq = q.shape[0], q.shape[1]
    args = _kv8_args(cache, page_table, pos0, None, T, q, writes=True)
    qp, q_stride = _rows3(q, "q", q.dtype)
    kp, k_stride = _rows3(k, "k", q.dtype, T, args[6])
    vp, v_stride = _rows3(v, "v", q.dtype, T, args[6])
    if hq == 0 or hq % args[6]:
        raise ValueError("%d query heads are not a multiple of %d kv heads" % (hq, args[6]))
    fp = 0
    if inv_freq is not None:
        fp = _chk(inv_freq, "inv_freq", torch.float32)
        if inv_freq.numel() < 64:
            raise ValueError("inv_freq must hold 64 values")
    for t in (k, v, inv_freq, out):
        if t is not None and t.device != q.device:
            raise ValueError("the tensors of a kv8 call lie on one device")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if args[12] else torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    else:
        if out.shape != q.shape:
            raise ValueError("out must be %s" % (tuple(q.shape),))
        _chk(out, "out", q.dtype)
        _disjoint(out, "out", q, k, v, *cache)
    S = args[12]
    scale = 128 ** -0.5 if scale is None else scale
    with torch.cuda.device(q.device):
        ws, ws_bytes, held = _kv8_workspace(workspace, S, T, T // S if S else 0, hq, args[6], q.device)
        call("ab200_kv8_step", qp, kp, vp, q_stride, k_stride, v_stride, out.data_ptr(), *args[:11], S, T, hq, 128, fp, float(scale), _code(q.dtype), ws, ws_bytes,
             _stream())
    return out


def kv_copy_pages(buffers, src, dst):
    """Copies the pages src[i] to dst[i] (host integers) inside every buffer [layers, pages, ...]: caches of any type, all in
    one launch.  A page's elements lie together.  No destination may occur twice or be a source too."""
    import ctypes
    if fast().kv_copy_pages(buffers, src, dst) is not None:
        return
    if len(src) != len(dst):
        raise ValueError("%d sources and %d destinations" % (len(src), len(dst)))
    buffers = list(buffers)
    if not buffers:
        raise ValueError("kv_copy_pages needs a buffer")
    pages, device = buffers[0].shape[1] if buffers[0].dim() >= 3 else 0, buffers[0].device
    base, layers, ls, ps, size = [], [], [], [], []
    for t in buffers:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError("a buffer must be a CUDA tensor (antares_b200 has no CPU path)")
        if t.dim() < 3 or t.shape[1] != pages or t.device != device or t.numel() == 0:
            raise ValueError("buffers must be [layers, pages, ...] with as many pages each, on one device; got %s" % (tuple(t.shape),))
        if not t[0, 0].is_contiguous():
            raise ValueError("the elements of a page must lie together")
        e = t.element_size()
        base.append(t.data_ptr())
        layers.append(t.shape[0])
        size.append(t[0, 0].numel() * e)
        ls.append(t.stride(0) * e if t.shape[0] > 1 else 0)
        ps.append(t.stride(1) * e if pages > 1 else size[-1])
    n, m, P = len(src), len(buffers), ctypes.c_void_p
    arr = lambda ty, v: ctypes.cast((ty * max(1, len(v)))(*v), P)  # noqa: E731
    with torch.cuda.device(device):
        call("ab200_kv_copy_pages", m, arr(P, base), arr(ctypes.c_int, layers), arr(ctypes.c_long, ls), arr(ctypes.c_long, ps), arr(ctypes.c_long, size), pages,
             arr(ctypes.c_int32, [int(i) for i in src]), arr(ctypes.c_int32, [int(i) for i in dst]), n, _stream())

"""Host-side operator surface of the grafted-SwiGLU path (Python mirror of
the reference's graft ops / layer / bake / norm / RoPE / optimizer entry
points), calling libglt.so through ctypes.

torch tensors are used only as device memory and for the current stream;
all arithmetic happens in the HIP kernels behind include/glt.h. Errors come
back as glt_amd._ffi.GltError (the reference throws std::runtime_error,
src/checks.hpp:10-18).
"""
import ctypes
import functools

import torch

from . import _ffi as F

PROJ_GATE, PROJ_UP, PROJ_DOWN = 0, 1, 2


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dtype_code(dtype):
    if dtype == torch.bfloat16:
        return F.DTYPE_BF16
    if dtype == torch.float32:
        return F.DTYPE_F32
    raise TypeError(f"unsupported dtype {dtype}")


def delta_offset(layer_idx, proj_idx, slice_dim, h_slice_dim):
    """Flat offset of (layer, projection) in [L*3, S, H] graft storage
    (reference src/graft_ops_impl.inc:5-7)."""
    return (layer_idx * 3 + proj_idx) * slice_dim * h_slice_dim


class GraftSlice:
    """One graft slice of one layer: placement + f32 masters [S,H] + the
    packed bf16 mirror (every orientation the GEMMs read; reference
    GraftWeights, src/types.hpp:190-201)."""

    def __init__(self, i_start, s, h_start, h, gate=None, up=None, down=None):
        self.i_start, self.s, self.h_start, self.h = int(i_start), int(s), int(h_start), int(h)
        self.gate, self.up, self.down = gate, up, down
        for t in (gate, up, down):
            if t is not None:
                assert t.dtype == torch.float32 and tuple(t.shape) == (self.s, self.h) and t.is_contiguous()
        dev = next(t.device for t in (gate, up, down) if t is not None) if any(
            t is not None for t in (gate, up, down)) else torch.device("cuda")
        nbytes = F.load().glt_graft_packed_size(self.s, self.h)
        self.packed = torch.zeros(nbytes // 2, dtype=torch.bfloat16, device=dev)

    def c_struct(self):
        return F.GraftSlice(self.i_start, self.s, self.h_start, self.h, _p(self.gate), _p(self.up), _p(self.down),
                            _p(self.packed))

    def pack(self):
        """Refresh the bf16 mirror from the masters (reference
        refresh_graft_weight_bf16, src/gemm_impl.inc:91-95)."""
        s = self.c_struct()
        F.call("glt_graft_pack", ctypes.byref(s), _p(self.packed), _stream())
        return self


def _slices_array(slices):
    arr = (F.GraftSlice * max(1, len(slices)))()
    for j, s in enumerate(slices):
        arr[j] = s.c_struct()
    return arr


class BaseMLP:
    """Frozen base weights of one MLP layer: gate/up [I,D], down [D,I], plus
    (bf16) the prepared copy the GEMMs read, made once."""

    def __init__(self, gate, up, down, prepare=True):
        self.gate, self.up, self.down = gate, up, down
        self.I, self.D = gate.shape
        self.dtype = gate.dtype
        self.prepared = None
        if prepare and self.I > 0:
            self.prepare()

    def prepare(self):
        d = F.MlpDesc(0, self.D, self.I, self.I, _dtype_code(self.dtype), 0, 0, None, None)
        nbytes = F.load().glt_base_prepared_size(ctypes.byref(d))
        if nbytes == 0:
            return self
        self.prepared = torch.empty(nbytes, dtype=torch.uint8, device=self.gate.device)
        F.call("glt_base_prepare", ctypes.byref(d), _p(self.gate), _p(self.up), _p(self.down), _p(self.prepared),
               _stream())
        return self

    def c_struct(self):
        return F.BaseWeights(_p(self.gate), _p(self.up), _p(self.down), _p(self.prepared))


def _desc(base, slices, M, N, explicit, recompute=False, state=None, residual=False, dy_f32=False, ckpt8=False):
    arr = _slices_array(slices)
    flags = ((F.MLP_EXPLICIT if explicit else 0) | (F.MLP_RECOMPUTE if recompute else 0)
             | (F.MLP_RESIDUAL if residual else 0) | (F.MLP_DY_F32 if dy_f32 else 0)
             | (F.MLP_SAVED_CKPT8 if ckpt8 else 0))
    d = F.MlpDesc(M, base.D, base.I, N, _dtype_code(base.dtype), flags, len(slices), arr,
                  ctypes.pointer(state) if state is not None else None)
    return d, arr


def mlp_forward(base, slices, x, N, explicit=True, save=True, residual=None):
    """Grafted SwiGLU forward (reference forward_layer FFN section,
    src/layer_forward_impl.inc:61-290). Returns y, gate_pre, up_pre, inter.
    With `residual` ([M,D], updated in place and returned as y) the output is
    added to it in the down GEMM's epilogue (reference x = x + ffn_out,
    src/layer_forward_impl.inc:271-275)."""
    M = x.shape[0]
    d, keep = _desc(base, slices, M, N, explicit, residual=residual is not None)
    y = residual if residual is not None else torch.empty((M, base.D), dtype=base.dtype, device=x.device)
    inter = torch.empty((M, N), dtype=base.dtype, device=x.device)
    g = torch.empty_like(inter) if save else None
    u = torch.empty_like(inter) if save else None
    b = base.c_struct()
    F.call("glt_mlp_fwd", ctypes.byref(d), ctypes.byref(b), _p(x), _p(y), _p(g), _p(u), _p(inter), _stream())
    return y, g, u, inter


def mlp_backward_workspace(base, slices, M, N, explicit=True, recompute=False, ckpt8=False):
    d, keep = _desc(base, slices, M, N, explicit, recompute, ckpt8=ckpt8)
    return F.load().glt_mlp_bwd_workspace_size(ctypes.byref(d))


def mlp_backward(base, slices, x, dy, N, gate_pre=None, up_pre=None, inter=None, want_dx=True, explicit=True,
                 recompute=False, state=None, workspace=None, norm=None, norm_in_place=False):
    """Graft-only backward (reference backward_layer FFN section,
    src/layer_backward_impl.inc:10-361). dy is [M,D] in the path dtype or
    f32 (the reference's upstream gradient, rounded once inside on the bf16
    path). Returns dx (f32) and per-slice [gate, up, down] f32 gradients in
    [S,H] storage. gate_pre and up_pre may be 8-bit checkpoints (ckpt8_save of
    the forward's); inter is then formed from them.

    norm = (norm_x, norm_w, var, eps): x is the output of that RMSNorm
    (reference rms_norm of the FFN input); the call then also runs its
    backward on dx (glt_mlp_rmsnorm_bwd, beside the weight-gradient GEMM)
    and returns (dx, grads, norm_dx); norm_in_place writes norm_dx over dx
    (the same tensor is returned twice)."""
    M = x.shape[0]
    if norm is not None:
        want_dx = True
    ckpt8 = isinstance(gate_pre, Ckpt8)
    if ckpt8:
        _need(isinstance(up_pre, Ckpt8) and (gate_pre.rows, gate_pre.cols) == (up_pre.rows, up_pre.cols) == (M, N),
              f"gate_pre and up_pre: checkpoints of [{M}, {N}]")
        gate_pre, up_pre = gate_pre.buf, up_pre.buf
    d, keep = _desc(base, slices, M, N, explicit, recompute, state, dy_f32=dy.dtype == torch.float32, ckpt8=ckpt8)
    nbytes = F.load().glt_mlp_bwd_workspace_size(ctypes.byref(d))
    if workspace is None or workspace.numel() < nbytes:
        workspace = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    dx = torch.empty((M, base.D), dtype=torch.float32, device=x.device) if want_dx else None
    grads = []
    garr = (F.GraftGrads * max(1, len(slices)))()
    for j, s in enumerate(slices):
        row = [torch.zeros((s.s, s.h), dtype=torch.float32, device=x.device) if t is not None else None
               for t in (s.gate, s.up, s.down)]
        grads.append(row)
        garr[j] = F.GraftGrads(_p(row[0]), _p(row[1]), _p(row[2]))
    b = base.c_struct()
    if norm is not None:
        norm_x, norm_w, var, eps = norm
        norm_dx = dx if norm_in_place else torch.empty((M, base.D), dtype=torch.float32, device=x.device)
        F.call("glt_mlp_rmsnorm_bwd", ctypes.byref(d), ctypes.byref(b), _p(x), _p(dy), _p(gate_pre), _p(up_pre),
               _p(inter), _p(dx), garr, _p(workspace), nbytes, _p(norm_x), _p(norm_w), _p(var), eps, _p(norm_dx),
               _stream())
        return dx, grads, norm_dx
    F.call("glt_mlp_bwd", ctypes.byref(d), ctypes.byref(b), _p(x), _p(dy), _p(gate_pre), _p(up_pre), _p(inter),
           _p(dx), garr, _p(workspace), nbytes, _stream())
    return dx, grads


class Ckpt8:
    """An activation [rows, cols] held in 8 bits for the backward: codes and an
    exponent per 32 columns in buf. Made by ckpt8_save."""

    def __init__(self, buf, rows, cols, dtype):
        self.buf, self.rows, self.cols, self.dtype = buf, rows, cols, dtype

    def load(self, dtype=None, out=None):
        """The values, bf16 or f32 (by default what was saved), into out where
        it is given."""
        buf, rows, cols = self.buf, self.rows, self.cols
        if out is None:
            out = torch.empty(rows, cols, dtype=dtype or self.dtype, device=buf.device)
        elif dtype not in (None, out.dtype) or out.shape != (rows, cols) or out.device != buf.device:
            raise ValueError(f"out: [{rows}, {cols}] on {buf.device}")
        dt, ld = _rows_ld("out", out)
        _call_on(buf, "glt_ckpt8_load", buf.data_ptr(), rows, cols, out.data_ptr(), dt, ld)
        return out


def _rows_ld(name, t):
    """(dtype code, row stride) of t [rows, cols] with contiguous rows."""
    rows, cols = t.shape
    ld, step = t.stride()
    if rows <= 1:
        ld = cols
    if (cols > 1 and step != 1) or ld < cols:
        raise ValueError(f"{name}: strides {t.stride()} (rows contiguous, not overlapping)")
    return _dtype_code(t.dtype), ld


@functools.lru_cache(maxsize=256)
def _ckpt8_size(rows, cols):
    return F.load().glt_ckpt8_size(rows, cols)


def ckpt8_save(x, buf=None):
    """x [rows, cols] bf16 or f32 as an 8-bit checkpoint, in buf (uint8,
    glt_ckpt8_size bytes) where it is given."""
    shape = x.shape
    _need(len(shape) == 2 and x.is_cuda, "x: [rows, cols] on a GPU")
    rows, cols = shape
    dt, ld = _rows_ld("x", x)
    buf = _workspace(buf, _ckpt8_size(rows, cols), x.device)
    _call_on(x, "glt_ckpt8_save", x.data_ptr(), dt, ld, rows, cols, buf.data_ptr())
    return Ckpt8(buf, rows, cols, x.dtype)


def ckpt8_swiglu(gate8, up8):
    """(gate, up, silu(gate) * up) bf16 [rows, cols] from checkpoints of the
    MLP's gate_pre and up_pre."""
    rows, cols, dev = gate8.rows, gate8.cols, gate8.buf.device
    _need((rows, cols) == (up8.rows, up8.cols) and up8.buf.device == dev, "gate8 and up8: checkpoints of one shape")
    gate, up, inter = (torch.empty(rows, cols, dtype=torch.bfloat16, device=dev) for _ in range(3))
    _call_on(gate8.buf, "glt_ckpt8_swiglu", gate8.buf.data_ptr(), up8.buf.data_ptr(), rows, cols, gate.data_ptr(),
             up.data_ptr(), inter.data_ptr())
    return gate, up, inter


def graft_gemm(kind, M, S, H, out, a=None, lda=0, delta=None, dy=None, ldo=None, alpha=1.0, beta=0.0):
    """One of the reference's six graft GEMM kinds (src/config.hpp:31-38)."""
    F.call("glt_graft_gemm", kind, M, S, H, _p(a), lda, _p(delta), _p(dy), _p(out),
           ldo if ldo is not None else out.shape[-1], alpha, beta, _stream())
    return out


def rms_norm(x, w, eps):
    """(y, variance) like the reference rms_norm (grafting.hip:116-146)."""
    M, D = x.shape
    y = torch.empty_like(x)
    var = torch.empty(M, dtype=torch.float32, device=x.device)
    F.call("glt_rmsnorm_fwd", _p(x), _p(w), _p(y), _p(var), M, D, eps, _stream())
    return y, var


def rms_norm_bwd(dy, x, w, var, eps, out=None):
    """Reference rms_norm_bwd (grafting.hip:153-172); dy f32, returns dx f32
    (into out when given, which may be dy itself)."""
    M, D = x.shape
    dx = torch.empty((M, D), dtype=torch.float32, device=x.device) if out is None else out
    F.call("glt_rmsnorm_bwd", _p(dy), _p(x), _p(w), _p(var), _p(dx), M, D, eps, _stream())
    return dx


def apply_rope(q, k, theta, pos_offset=0):
    """In-place RoPE on q [B,T,nq,hd] and k [B,T,nk,hd], dense bf16 (reference
    apply_rope, src/rope_impl.inc:8-39). It has no backward: the gradients of
    attention_bwd are those on the rotated q and k."""
    for name, t in (("q", q), ("k", k)):
        _need(t is None or t.is_contiguous(), f"{name}: contiguous (parts of a fused projection are not)")
    B, T, nq, hd = q.shape
    nk = k.shape[2] if k is not None else 0
    F.call("glt_rope_fwd", _p(q), nq, _p(k), nk, B, T, hd, theta, pos_offset, _stream())


def attention(q, k, v, causal=True, scale=None):
    """Causal GQA attention forward (the reference's SDPA call in
    forward_layer, src/layer_forward_impl.inc:41-49). q [B,T,Hq,hd],
    k/v [B,T,Hkv,hd] dense bf16; returns [B,T,Hq,hd]. (attention_train takes
    parts of a fused projection.)"""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _need(t.is_contiguous(), f"{name}: contiguous (parts of a fused projection are not)")
    B, T, Hq, hd = q.shape
    Hkv = k.shape[2]
    if scale is None:
        scale = hd ** -0.5
    out = torch.empty_like(q)
    nb = F.load().glt_attention_workspace_size(B, T, Hkv, hd)
    ws = torch.empty(nb, dtype=torch.uint8, device=q.device)
    F.call("glt_attention_fwd", _p(q), _p(k), _p(v), _p(out), B, T, Hq, Hkv, hd, scale, 1 if causal else 0,
           _p(ws), nb, _stream())
    return out


def _need(cond, msg):
    if not cond:
        raise ValueError(msg)


def _workspace(ws, nbytes, device):
    """ws where it is given (uint8, on the device, at least nbytes), else a new one."""
    if ws is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    if ws.dtype != torch.uint8 or ws.device != device or not ws.is_contiguous() or ws.numel() < nbytes:
        raise ValueError(f"workspace: {nbytes} contiguous uint8 on {device}")
    return ws


def _a(t):
    """A tensor's address (ctypes takes it for a pointer as it is)."""
    return None if t is None else t.data_ptr()


# the current stream's handle by device index (the Stream object that the public
# function makes first costs 2 us of a small call's 12)
_stream_handle = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call_on(t, name, *args):
    """The entry point on t's device and that device's current stream, which
    is passed last."""
    index = t.get_device()
    if index == torch.cuda.current_device():
        F.check(getattr(F.load(), name)(*args, _stream_handle(index)), name)
    else:
        with torch.cuda.device(index):
            F.call(name, *args, _stream_handle(index))


def _heads_ld(name, t, B, T, device):
    """Elements between the tokens of t [B, T, heads, head_dim]; heads lie
    next to each other, sequences T tokens apart."""
    shape = t.shape
    if len(shape) != 4 or shape[0] != B or shape[1] != T or t.dtype != torch.bfloat16 or t.device != device:
        raise ValueError(f"{name}: bf16 [{B}, {T}, heads, head_dim] on {device}, not {t.dtype} {tuple(shape)} on "
                         f"{t.device}")
    H, hd = shape[2], shape[3]
    sb, st, sh, se = t.stride()
    if se == 1 and sh == hd and st >= H * hd > 0 and sb == T * st:  # as they mostly come
        return st
    if B * T == 0:
        return H * hd
    ld = st if T > 1 else sb if B > 1 else H * hd
    if (hd > 1 and se != 1) or (H > 1 and sh != hd) or (B > 1 and sb != T * ld):
        raise ValueError(f"{name}: strides {t.stride()} (a token's heads contiguous, tokens evenly spaced)")
    return ld


def _check_window(window, sinks):
    if window is None:
        _need(sinks == 0, "sinks: with a window")
    elif not (1 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31):
        raise ValueError(f"window {window} (None, or 1 to 2^31 - 1), sinks {sinks}")


def _attn_train_desc(q, k, v, out, causal, scale, seq_lens):
    """out None: a new dense one."""
    shape = q.shape
    _need(len(shape) == 4 and q.is_cuda, "q: [B, T, heads, head_dim] on a GPU")
    B, T, Hq, hd = shape
    dev = q.device
    lds = (_heads_ld("q", q, B, T, dev), _heads_ld("k", k, B, T, dev), _heads_ld("v", v, B, T, dev),
           Hq * hd if out is None else _heads_ld("out", out, B, T, dev))
    kshape = k.shape
    _need(kshape == v.shape and kshape[3] == hd and (out is None or out.shape == shape), "k, v and out do not fit q")
    if seq_lens is not None and not (seq_lens.dtype == torch.int32 and seq_lens.shape == (B,)
                                     and seq_lens.device == dev and seq_lens.is_contiguous()):
        raise ValueError(f"seq_lens: contiguous int32 [{B}] on {dev}")
    d = F.AttnDesc(B, T, Hq, kshape[2], hd, hd ** -0.5 if scale is None else scale, 1 if causal else 0, *lds,
                   _a(seq_lens))
    return d, (B, T, Hq, kshape[2], hd), lds


def attention_train(q, k, v, causal=True, scale=None, seq_lens=None, window=None, sinks=0):
    """GQA attention forward of a training step: (out [B,T,Hq,hd] bf16, lse
    [B,Hq,T] f32) for attention_bwd. q [B,T,Hq,hd], k/v [B,T,Hkv,hd] bf16, also
    as views of one projection output [B,T,(Hq+2Hkv)*hd]. seq_lens int32 [B]:
    the lengths of a padded batch (rows past them: zero output, lse -inf).
    window=W: of the keys up to itself a row reads the last W (its own among
    them) and the first `sinks` of its sequence (up to 1024 where W < T)."""
    _check_window(window, sinks)
    d, (B, T, Hq, _, _), _ = _attn_train_desc(q, k, v, None, causal, scale, seq_lens)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device)
    name, sight = ("glt_attention_train_fwd", ()) if window is None else ("glt_attention_window_fwd", (window, sinks))
    _call_on(q, name, ctypes.byref(d), *sight, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr())
    return out, lse


@functools.lru_cache(maxsize=256)
def _attention_bwd_size(B, T, Hq, Hkv, hd, window=0, sinks=0):
    return F.load().glt_attention_window_bwd_workspace_size(ctypes.byref(F.AttnDesc(B, T, Hq, Hkv, hd)), window, sinks)


def _attn_grad_buffers(q, k, v, shape, lds):
    """Gradients with the strides of q, k, v: parts of one buffer where q, k, v
    are parts of one (that do not overlap)."""
    B, T, Hq, Hkv, hd = shape
    ld, k_ld, v_ld, _ = lds
    rows, nq, nk = B * T, 2 * hd * Hq, 2 * hd * Hkv  # nq, nk: bytes of a token's heads
    if ld == Hq * hd and k_ld == v_ld == Hkv * hd and rows > 1:  # dense, as they mostly come
        return [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v)]
    if ld == k_ld == v_ld:
        pq, pk, pv = q.data_ptr(), k.data_ptr(), v.data_ptr()
        (p0, n0), (p1, n1), (p2, n2) = sorted(((pq, nq), (pk, nk), (pv, nk)))
        if p0 + n0 <= p1 and p1 + n1 <= p2 and p2 + n2 <= p0 + 2 * ld:
            buf = torch.empty(rows * ld, dtype=q.dtype, device=q.device)
            strides = (T * ld, ld, hd, 1)
            return [buf.as_strided(t.shape, strides, (p - p0) // 2) for p, t in ((pq, q), (pk, k), (pv, v))]
    return [torch.empty(rows * n, dtype=q.dtype, device=q.device).as_strided(t.shape, (T * n, n, hd, 1))
            for t, n in ((q, ld), (k, k_ld), (v, v_ld))]


def attention_bwd(q, k, v, out, lse, dout, causal=True, scale=None, seq_lens=None, grads=None, workspace=None, window=None,
                  sinks=0):
    """(dq, dk, dv) of attention_train (with its window and sinks), bf16 with the strides of q, k, v (parts
    of one buffer where q, k, v are; `grads` gives them, overlapping no input).
    out and lse are the forward's; dout has out's shape and strides. workspace: a uint8 tensor of
    glt_attention_bwd_workspace_size (glt_attention_window_bwd_workspace_size) bytes to use instead of a new one."""
    _check_window(window, sinks)
    d, shape, lds = _attn_train_desc(q, k, v, out, causal, scale, seq_lens)
    B, T, Hq, _, _ = shape
    dev = q.device
    _need(_heads_ld("dout", dout, B, T, dev) == lds[3] and dout.shape == out.shape, "dout: out's shape and strides")
    if lse.dtype != torch.float32 or lse.shape != (B, Hq, T) or not lse.is_contiguous() or lse.device != dev:
        raise ValueError(f"lse: contiguous f32 [{B}, {Hq}, {T}] on {dev}")
    if grads is None:
        grads = _attn_grad_buffers(q, k, v, shape, lds)
    else:
        for n, t, x, ld in zip(("dq", "dk", "dv"), grads, (q, k, v), lds):
            _need(t.shape == x.shape and _heads_ld(n, t, B, T, dev) == ld, "dq, dk, dv: the shapes and strides of q, k, v")
    name, sight = ("glt_attention_bwd", ()) if window is None else ("glt_attention_window_bwd", (window, sinks))
    workspace = _workspace(workspace, _attention_bwd_size(*shape, *sight), dev)
    dq, dk, dv = grads
    _call_on(q, name, ctypes.byref(d), *sight, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
             lse.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), workspace.data_ptr(),
             workspace.numel())
    return dq, dk, dv


def _table_ld(name, t, rows, index):
    """Elements between the rows of a page table int32 [rows, pages]."""
    shape = t.shape
    if t.dtype is not torch.int32 or len(shape) != 2 or shape[0] != rows or t.get_device() != index:
        raise ValueError(f"{name}: int32 [{rows}, pages] on GPU {index}")
    n = shape[1]
    ld, step = t.stride()
    if step == 1 and ld >= n:
        return ld
    if (n > 1 and step != 1) or (rows > 1 and n != 0):
        raise ValueError(f"{name}: strides {t.stride()} (a row's pages contiguous, rows apart)")
    return n


def _check_ints(name, t, n, index):
    if t.dtype is not torch.int32 or t.shape != (n,) or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 [{n}] on GPU {index}")


class Kv8Cache:
    """The keys and values of one layer in 8 bits, for generation: n_pages pages
    of 64 tokens, n_kv_heads heads of 128 (glt_kv8_cache). Sequence b of a call
    holds lens[b] tokens, of which token i lies in page pages[b, i // 64]; the
    call's new tokens are its last new_lens[b] (None: T). pages int32 [B, n],
    lens and new_lens int32 [B], on the cache's device. What keeps the tables,
    and which page is free, is the caller's."""

    PAGE = 64

    def __init__(self, n_pages, n_kv_heads, head_dim=128, device="cuda"):
        nbytes = F.load().glt_kv8_size(n_pages, n_kv_heads, head_dim)
        _need(nbytes > 0, f"Kv8Cache: {n_pages} pages of {n_kv_heads} heads of {head_dim} (head_dim 128)")
        self.data = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _need(self.data.is_cuda, "Kv8Cache: a GPU device")
        self.n_pages, self.n_kv_heads, self.head_dim = n_pages, n_kv_heads, head_dim
        self._index, self._device = self.data.get_device(), self.data.device
        self._heads = (n_kv_heads, head_dim)
        self._c = F.Kv8Cache(self.data.data_ptr(), n_pages, n_kv_heads, head_dim)
        self._ref = ctypes.byref(self._c)

    def _seqs(self, B, T, pages, lens, new_lens):
        index = self._index
        ld = _table_ld("pages", pages, B, index)
        _check_ints("lens", lens, B, index)
        if new_lens is not None:
            _check_ints("new_lens", new_lens, B, index)
            new_lens = new_lens.data_ptr()
        return F.Kv8Seqs(B, T, pages.data_ptr(), ld, pages.shape[1], lens.data_ptr(), new_lens)

    def write(self, k, v, pages, lens, new_lens=None):
        """The new tokens' k and v [B, T, n_kv_heads, 128] bf16, also as views of
        one projection output, into the cache."""
        self._tokens("glt_kv8_write", k, v, pages, lens, new_lens)

    def read(self, pages, lens, T, new_lens=None, out=None):
        """(k, v) bf16 [B, T, n_kv_heads, 128] of the last new_lens[b] (None: T)
        tokens, into `out` where it is given; zeros past them."""
        if out is None:
            k = torch.empty((pages.shape[0], T, *self._heads), dtype=torch.bfloat16, device=self._device)
            out = k, torch.empty_like(k)
        elif out[0].shape[:2] != (pages.shape[0], T):
            raise ValueError(f"out: {pages.shape[0]} x {T} tokens")
        self._tokens("glt_kv8_read", *out, pages, lens, new_lens)
        return out

    def _tokens(self, name, k, v, pages, lens, new_lens):
        shape = k.shape
        if len(shape) != 4 or shape[2:] != self._heads or shape != v.shape:
            raise ValueError(f"k, v: [B, T, {self.n_kv_heads}, {self.head_dim}]")
        B, T, _, _ = shape
        dev = self._device
        k_ld, v_ld = _heads_ld("k", k, B, T, dev), _heads_ld("v", v, B, T, dev)
        s = self._seqs(B, T, pages, lens, new_lens)
        _call_on(self.data, name, self._ref, ctypes.byref(s), k.data_ptr(), k_ld, v.data_ptr(), v_ld)

    def attention(self, q, pages, lens, new_lens=None, scale=None, window=None, sinks=0, prefix=None, workspace=None):
        """Attention of the new tokens q [B, T, Hq, 128] bf16 (written before)
        over the cache: (out [B, T, Hq, 128] bf16, lse [B, Hq, T] f32). Token p
        reads tokens j <= p, of which window=W leaves j > p - W and the first
        `sinks` (0 without a window). prefix = (pages int32 [groups, m], lens int32 [groups]): each
        group of B / groups consecutive sequences continues these tokens, which are
        read once for the group. Rows past new_lens: zeros and -inf. workspace: a
        uint8 tensor of glt_kv8_attention_workspace_size bytes instead of a new
        one."""
        shape = q.shape
        if len(shape) != 4 or shape[3] != self.head_dim:
            raise ValueError(f"q: [B, T, heads, {self.head_dim}]")
        B, T, Hq, hd = shape
        dev, index = self._device, self._index
        q_ld = _heads_ld("q", q, B, T, dev)
        _check_window(window, sinks)
        s = self._seqs(B, T, pages, lens, new_lens)
        d = F.Kv8Attn(Hq, hd ** -0.5 if scale is None else scale, window or 0, sinks)
        if prefix is not None:
            ppages, plens = prefix
            groups = d.n_groups = ppages.shape[0]
            _need(groups > 0 or B == 0, "prefix: no groups")
            d.prefix_ld = _table_ld("prefix pages", ppages, groups, index)
            _check_ints("prefix lens", plens, groups, index)
            d.prefix_pages, d.n_prefix_table, d.prefix_lens = ppages.data_ptr(), ppages.shape[1], plens.data_ptr()
        refs = self._ref, ctypes.byref(s), ctypes.byref(d)
        nbytes = F.load().glt_kv8_attention_workspace_size(*refs)
        if nbytes:
            workspace = _workspace(workspace, nbytes, dev)
            ws = workspace.data_ptr(), workspace.numel()
        else:  # one launch: nothing between
            ws = None, 0
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty((B, Hq, T), dtype=torch.float32, device=dev)
        _call_on(self.data, "glt_kv8_attention", *refs, q.data_ptr(), q_ld, out.data_ptr(), Hq * hd, lse.data_ptr(), *ws)
        return out, lse


def adamw_step(w, g, m, v, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, clip_norm=0.0,
               mirror=None):
    """One AdamW step (reference adamw_fused_kernel + optional global clip)."""
    n = w.numel()
    ws_bytes = F.load().glt_adamw_workspace_size(n)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=w.device) if clip_norm > 0 else None
    F.call("glt_adamw_step", _p(w), _p(g), _p(m), _p(v), _p(mirror), n, step, lr, beta1, beta2, eps, weight_decay,
           clip_norm, _p(ws), ws_bytes if ws is not None else 0, _stream())


def adamw_graft_step(slices, grads, m, v, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01,
                     proj_mask=7, clip_norm=0.0, workspace=None):
    """AdamW over graft slices with the packed-mirror refresh fused in and
    the optional global-L2 clip over all of their gradients (reference
    grafting.hip:1149-1164, clip 1.0 by default there).
    grads/m/v: per slice a flat f32 [3*S*H] tensor (gate, up, down)."""
    arr = _slices_array(slices)
    nbytes = F.load().glt_adamw_workspace_size(0)
    if clip_norm > 0 and workspace is None:
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=grads[0].device)
    F.call("glt_adamw_graft_step", arr, len(slices), F.ptr_array([g.data_ptr() for g in grads]),
           F.ptr_array([t.data_ptr() for t in m]), F.ptr_array([t.data_ptr() for t in v]),
           F.ptr_array([s.packed.data_ptr() for s in slices]), proj_mask, step, lr, beta1, beta2, eps,
           weight_decay, clip_norm, _p(workspace), nbytes if workspace is not None else 0, _stream())


def shadow_bake(state, gate, up, down, grafts, placements, *, D, I, N=None, materialize=False, gate_out=None,
                up_out=None, down_out=None, layer_start=0, layer_end=None, proj_mask=7, graft_dtype=None):
    """Bake graft deltas into bf16 base matrices (reference
    apply_graft_to_shadow, src/shadow_bake_impl.inc:58-128).

    gate/up/down: per-layer lists of bf16 tensors; grafts[j][l]: slice j's
    flat [3,S,H] deltas for layer l; placements[j] = (i0, S, h0, H)."""
    L = len(gate)
    n_sl = len(placements)
    if graft_dtype is None:
        graft_dtype = grafts[0][0].dtype if n_sl else torch.float32
    pl = (ctypes.c_int32 * max(1, 4 * n_sl))(*[int(v) for p in placements for v in p])
    gptr = F.ptr_array([grafts[j][l].data_ptr() for j in range(n_sl) for l in range(L)])
    d = F.BakeDesc(F.BAKE_MATERIALIZE if materialize else F.BAKE_IN_PLACE, L, layer_start,
                   L - 1 if layer_end is None else layer_end, proj_mask, D, I, N if N is not None else I,
                   _dtype_code(graft_dtype), n_sl, pl, gptr)

    def arr(ts):
        return F.ptr_array([t.data_ptr() for t in ts]) if ts is not None else None

    F.call("glt_shadow_bake", ctypes.byref(d), ctypes.byref(state), arr(gate), arr(up), arr(down), arr(gate_out),
           arr(up_out), arr(down_out), _stream())


def f32_to_bf16(x):
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    F.call("glt_f32_to_bf16", _p(x), _p(out), x.numel(), _stream())
    return out


def fill_normal(t, seed, tensor_id, mean=0.0, std=1.0):
    F.call("glt_fill_normal", _p(t), _dtype_code(t.dtype), t.numel(), seed, tensor_id, mean, std, _stream())
    return t


def silu_mul(g, u):
    out = torch.empty_like(g)
    F.call("glt_silu_mul", _p(g), _p(u), _p(out), g.numel(), _stream())
    return out


def gate_up_bwd(gi, g, u):
    dg = torch.empty(gi.shape, dtype=torch.float32, device=gi.device)
    du = torch.empty_like(dg)
    F.call("glt_gate_up_bwd", _p(gi), _p(g), _p(u), _p(dg), _p(du), gi.numel(), _stream())
    return dg, du


class DecoderLayer:
    """One decoder layer with the grafted MLP (reference forward_layer,
    src/layer_forward_impl.inc:15-290) over glt_layer_fwd. Projection weights
    bf16 [out, in]; base is the MLP's BaseMLP; slices its graft slices."""

    def __init__(self, B, T, n_q_heads, n_kv_heads, wq, wk, wv, wo, ln_in, ln_post, base, slices, N,
                 rope_theta=500000.0, rms_eps=1e-5, explicit=True, head_dim=128):
        self.base, self.slices = base, slices
        md, self._keep = _desc(base, slices, B * T, N, explicit)
        self.desc = F.LayerDesc(B, T, n_q_heads, n_kv_heads, head_dim, rope_theta, rms_eps, md)
        self._w = (wq, wk, wv, wo, ln_in, ln_post)
        self.prepared = torch.empty(F.load().glt_attn_prepared_size(ctypes.byref(self.desc)), dtype=torch.uint8,
                                    device=wq.device)
        self.weights = F.LayerWeights(_p(wq), _p(wk), _p(wv), _p(wo), _p(ln_in), _p(ln_post), _p(self.prepared),
                                      base.c_struct())
        F.call("glt_attn_prepare", ctypes.byref(self.desc), ctypes.byref(self.weights), _p(self.prepared), _stream())
        self.ws = torch.empty(F.load().glt_layer_fwd_workspace_size(ctypes.byref(self.desc)), dtype=torch.uint8,
                              device=wq.device)

    def forward(self, x, inter=None):
        """x [B*T, D] bf16, updated in place; returns (x, x_ffn, ffn_var)."""
        M, D = x.shape
        x_ffn = torch.empty_like(x)
        var = torch.empty(M, dtype=torch.float32, device=x.device)
        F.call("glt_layer_fwd", ctypes.byref(self.desc), ctypes.byref(self.weights), _p(x), _p(x_ffn), _p(var),
               None, None, _p(inter), _p(self.ws), self.ws.numel(), _stream())
        return x, x_ffn, var


def _grft_info(num_layers, S, H, hidden_dim=0, domain_id=0, session_id=""):
    return F.GrftInfo(num_layers, S, H, hidden_dim, domain_id, session_id.encode() if session_id else None)


def grft_save(path, weight, num_layers, S, H, hidden_dim=0, domain_id=0, session_id=""):
    """Writes the flat f32 graft storage [num_layers*3*S*H] (device or host
    tensor) as a GRFT checkpoint (reference save_safetensors,
    src/checkpoint_impl.inc:39-97)."""
    info = _grft_info(num_layers, S, H, hidden_dim, domain_id, session_id)
    F.call("glt_grft_save", str(path).encode(), ctypes.byref(info), _p(weight), int(weight.is_cuda),
           _stream() if weight.is_cuda else None)


def grft_load(path, weight, num_layers, S, H, domain_id=0, session_id="", raw_f32=False):
    """Loads a GRFT checkpoint (reference load_safetensors_checkpoint,
    src/checkpoint_impl.inc:170-285) or, with raw_f32, an --init-deltas file
    into the f32 storage tensor `weight` (device or host)."""
    info = _grft_info(num_layers, S, H, 0, domain_id, session_id)
    F.call("glt_grft_load_raw_f32" if raw_f32 else "glt_grft_load", str(path).encode(), ctypes.byref(info),
           _p(weight), int(weight.is_cuda), _stream() if weight.is_cuda else None)
    return weight

def masked_ce(logits, ids, ood=None, scale=1.0, grad=None, want_grad=True, ce_per_token=False):
    """Masked cross-entropy over the shifted logits and its gradient
    (reference loss grafting.hip:1027-1050, grad_logits :1122-1135).
    logits [B,T,V] bf16, ids [B,T] int32, ood [B,T] int32 or None.
    Returns (stats [loss, target-logit mean, target-prob mean, n] f32 on the
    device, grad [B,T,V] bf16 or None, ce [B*(T-1)] f32 or None). Pass
    grad=logits to overwrite the logits with the gradient."""
    B, T, V = logits.shape
    dev = logits.device
    stats = torch.empty(4, dtype=torch.float32, device=dev)
    if want_grad and grad is None:
        grad = torch.empty_like(logits)
    ce = torch.empty(max(B * (T - 1), 1), dtype=torch.float32, device=dev) if ce_per_token else None
    nbytes = F.load().glt_masked_ce_workspace_size(B, T)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    F.call("glt_masked_ce", _p(logits), logits.stride(1), _p(ids), _p(ood), B, T, V, scale,
           _p(grad) if want_grad else None, grad.stride(1) if want_grad else 0, _p(ce), _p(stats), _p(ws), nbytes,
           _stream())
    return stats, (grad if want_grad else None), ce


def _logit_rows(logits, ids):
    """(rows, V, row stride, dtype code) of logits [rows, V], bf16 or f32;
    checks ids [rows, n] int32."""
    _need(logits.dim() == 2 and logits.is_cuda, "logits: [rows, V] on a GPU")
    rows, V = logits.shape
    dt = _dtype_code(logits.dtype)
    ld = logits.stride(0) if rows > 1 else V
    if (V > 1 and logits.stride(1) != 1) or ld < V:
        raise ValueError(f"logits: strides {logits.stride()} (rows contiguous, not overlapping)")
    if ids is not None and not (ids.dim() == 2 and ids.shape[0] == rows and ids.dtype == torch.int32
                                and ids.device == logits.device and ids.is_contiguous()):
        raise ValueError(f"ids: contiguous int32 [{rows}, n] on {logits.device}")
    return rows, V, ld, dt


def _row_values(name, t, shape, device):
    if t.dtype != torch.float32 or tuple(t.shape) != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous f32 {list(shape)} on {device}")


@functools.lru_cache(maxsize=256)
def _logprobs_size(rows, V, dt, top_k):
    return F.load().glt_token_logprobs_workspace_size(rows, V, dt, top_k)


def token_logprobs(logits, ids=None, top_k=0, temperature=1.0, workspace=None):
    """Log probabilities under softmax(logits / temperature) of the given
    tokens ids [rows, n] int32 (below 0 = padding, 0), with what else an answer
    shows of each row: dict(logprobs [rows, n], entropy [rows], lse [rows]) and,
    with top_k, top_ids int32 and top_logprobs [rows, top_k]. logits [rows, V]
    bf16 or f32."""
    rows, V, ld, dt = _logit_rows(logits, ids)
    dev = logits.device
    n = ids.shape[1] if ids is not None else 0
    f32, empty = torch.float32, torch.empty
    logprobs = empty(rows, n, dtype=f32, device=dev)
    entropy, lse = empty(rows, dtype=f32, device=dev), empty(rows, dtype=f32, device=dev)
    r = dict(logprobs=logprobs, entropy=entropy, lse=lse)
    top_ids = top_logprobs = None
    if top_k > 0:
        r["top_ids"] = top_ids = empty(rows, top_k, dtype=torch.int32, device=dev)
        r["top_logprobs"] = top_logprobs = empty(rows, top_k, dtype=f32, device=dev)
    ws = _workspace(workspace, _logprobs_size(rows, V, dt, top_k), dev)
    _call_on(logits, "glt_token_logprobs", _a(logits), dt, ld, rows, V, temperature, _a(ids), n, top_k,
             logprobs.data_ptr(), entropy.data_ptr(), lse.data_ptr(), _a(top_ids), _a(top_logprobs), ws.data_ptr(),
             ws.numel())
    return r


def token_logprobs_bwd(logits, ids, lse, grad_logprobs, entropy=None, grad_entropy=None, temperature=1.0, grad=None):
    """Gradient on the logits (their dtype) of sum(grad_logprobs * logprobs) +
    sum(grad_entropy * entropy), from token_logprobs' lse and entropy. Pass
    grad=logits to overwrite the logits with it."""
    rows, V, ld, dt = _logit_rows(logits, ids)
    dev = logits.device
    n = ids.shape[1] if ids is not None else 0
    _row_values("lse", lse, (rows,), dev)
    if n:
        _row_values("grad_logprobs", grad_logprobs, (rows, n), dev)
    if grad_entropy is not None:
        _need(entropy is not None, "grad_entropy needs the forward's entropy")
        _row_values("grad_entropy", grad_entropy, (rows,), dev)
        _row_values("entropy", entropy, (rows,), dev)
    if grad is None:
        grad = torch.empty((rows, V), dtype=logits.dtype, device=dev)
    _need(grad.shape == logits.shape and grad.dtype == logits.dtype and grad.device == dev
          and (V == 1 or grad.stride(1) == 1), "grad: the logits' shape, dtype and device, rows contiguous")
    _call_on(logits, "glt_token_logprobs_bwd", _a(logits), dt, ld, rows, V, temperature, _a(ids), n,
             _a(grad_logprobs if n else None), _a(lse), _a(entropy if grad_entropy is not None else None),
             _a(grad_entropy), _a(grad), grad.stride(0) if rows > 1 else V)
    return grad


def silence_energy(delta, ld=None):
    """Per-token energy ||delta_t|| / sqrt(slice) of [tokens, slice] f32 or
    bf16 rows (reference compute_energy_kernel)."""
    tokens, slice_ = delta.shape
    out = torch.empty(tokens, dtype=torch.float32, device=delta.device)
    dt = F.DTYPE_F32 if delta.dtype == torch.float32 else F.DTYPE_BF16
    F.call("glt_silence_energy", _p(delta), dt, ld if ld is not None else delta.stride(0), tokens, slice_, _p(out),
           _stream())
    return out


def silence_blend(dy, delta, ood, lam):
    """In place: dy += lam * delta / (||delta|| sqrt(slice)) on OOD tokens
    (reference silence_blend_kernel)."""
    tokens, slice_ = delta.shape
    F.call("glt_silence_blend", _p(dy), _p(delta), _p(ood), tokens, slice_, lam, _stream())
    return dy


def silence_blend_energy(dy_gate, delta_gate, dy_up, delta_up, ood, lam, energies=True):
    """Gate and up silence blend with their energies (reference
    fused_silence_blend_energy_kernel); returns (energy_gate, energy_up)."""
    tokens, slice_ = delta_gate.shape
    eg = torch.empty(tokens, dtype=torch.float32, device=dy_gate.device) if energies else None
    eu = torch.empty(tokens, dtype=torch.float32, device=dy_gate.device) if energies else None
    F.call("glt_silence_blend_energy", _p(dy_gate), _p(delta_gate), _p(dy_up), _p(delta_up), _p(eg), _p(eu), _p(ood),
           tokens, slice_, lam, _stream())
    return eg, eu


def lr_schedule(step, total_steps, warmup_steps, lr_peak):
    """Warmup + cosine learning rate (reference get_lr, src/config.hpp:122-129)."""
    return F.load().glt_lr_schedule(step, total_steps, warmup_steps, lr_peak)


class SafetensorsModel:
    """Base-model weights in safetensors files (reference
    load_base_model_safetensors, src/model_io_impl.inc:57-190): a file or a
    directory of *.safetensors, memory-mapped by the library."""

    def __init__(self, path):
        self._h = ctypes.c_void_p()
        F.call("glt_st_open", str(path).encode(), ctypes.byref(self._h))

    def close(self):
        if self._h:
            F.load().glt_st_close(self._h)
            self._h = ctypes.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __len__(self):
        return F.load().glt_st_count(self._h)

    def info(self, name):
        """(dtype code, shape) of tensor `name`."""
        dt, nd = ctypes.c_int32(), ctypes.c_int32()
        shape = (ctypes.c_int64 * 8)()
        F.call("glt_st_info", self._h, name.encode(), ctypes.byref(dt), ctypes.byref(nd), shape)
        return dt.value, tuple(shape[i] for i in range(nd.value))

    def read(self, name, dtype=torch.bfloat16, transpose=False, device="cuda"):
        """Tensor `name` as bf16 or f32, optionally transposed (2-D)."""
        _, shape = self.info(name)
        if transpose:
            shape = shape[::-1]
        out = torch.empty(shape, dtype=dtype, device=device)
        on_dev = out.is_cuda
        F.call("glt_st_read", self._h, name.encode(), _p(out), F.DTYPE_F32 if dtype == torch.float32 else F.DTYPE_BF16,
               int(transpose), int(on_dev), _stream() if on_dev else None)
        return out

    def load_layer(self, layer, D, I, n_q_heads, n_kv_heads, head_dim, device="cuda"):
        """The nine bf16 weights of decoder layer `layer` (names and shapes of
        the reference's loader); returns a dict."""
        nq, nk = n_q_heads * head_dim, n_kv_heads * head_dim
        shapes = {"q_proj": (nq, D), "k_proj": (nk, D), "v_proj": (nk, D), "o_proj": (D, nq), "ln_in": (D,),
                  "ln_post": (D,), "gate": (I, D), "up": (I, D), "down": (D, I)}
        out = {k: torch.empty(v, dtype=torch.bfloat16, device=device) for k, v in shapes.items()}
        bufs = F.LayerBuffers(*[out[k].data_ptr() for k in shapes])
        md = F.MlpDesc(1, D, I, I, F.DTYPE_BF16, 0, 0, None, None)
        ld = F.LayerDesc(1, 1, n_q_heads, n_kv_heads, head_dim, 0.0, 1e-5, md)
        on_dev = torch.device(device).type == "cuda"
        F.call("glt_st_load_layer", self._h, layer, ctypes.byref(ld), ctypes.byref(bufs), int(on_dev),
               _stream() if on_dev else None)
        return out

    def load_head(self, V, D, device="cuda"):
        """(embed [V,D], final norm [D], lm_head [V,D]) as bf16; lm_head tied
        to the embedding when the files have none."""
        embed = torch.empty((V, D), dtype=torch.bfloat16, device=device)
        norm = torch.empty(D, dtype=torch.bfloat16, device=device)
        head = torch.empty((V, D), dtype=torch.bfloat16, device=device)
        on_dev = embed.is_cuda
        F.call("glt_st_load_head", self._h, V, D, _p(embed), _p(norm), _p(head), int(on_dev),
               _stream() if on_dev else None)
        return embed, norm, head


class Model:
    """forward_model (reference grafting.hip:224-271) over DecoderLayer
    objects: embedding, the layers, final RMSNorm, LM head. embed / lm_head
    [V,D] bf16, final_norm [D] bf16."""

    def __init__(self, layers, embed, final_norm, lm_head=None):
        self.layers = layers
        self.embed, self.final_norm = embed, final_norm
        self.lm_head = embed if lm_head is None else lm_head      # tied when absent
        self.V, self.D = self.lm_head.shape
        lib = F.load()
        self.lm_prepared = torch.empty(lib.glt_lm_head_prepared_size(self.V, self.D), dtype=torch.uint8,
                                       device=self.lm_head.device)
        F.call("glt_lm_head_prepare", _p(self.lm_head), self.V, self.D, _p(self.lm_prepared), _stream())
        n = len(layers)
        self._descs = (F.LayerDesc * n)(*[l.desc for l in layers])
        self._weights = (F.LayerWeights * n)(*[l.weights for l in layers])

    def _c(self, explicit):
        return F.Model(len(self.layers), self.V, int(explicit), self._descs, self._weights, _p(self.embed),
                       _p(self.final_norm), _p(self.lm_head), _p(self.lm_prepared))

    def forward(self, ids, explicit=True):
        """ids [B,T] int32 on the device; returns logits [B*T, V] bf16."""
        m = self._c(explicit)
        M = ids.numel()
        logits = torch.empty((M, self.V), dtype=torch.bfloat16, device=ids.device)
        nbytes = F.load().glt_model_fwd_workspace_size(ctypes.byref(m))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=ids.device)
        F.call("glt_model_fwd", ctypes.byref(m), _p(ids), _p(logits), _p(ws), nbytes, _stream())
        return logits


def lm_head_fwd(x, lm_head, prepared=None):
    """logits [M,V] = x [M,D] . lm_head^T (at::linear), bf16."""
    V, D = lm_head.shape
    if prepared is None:
        prepared = torch.empty(F.load().glt_lm_head_prepared_size(V, D), dtype=torch.uint8, device=x.device)
        F.call("glt_lm_head_prepare", _p(lm_head), V, D, _p(prepared), _stream())
    out = torch.empty((x.shape[0], V), dtype=torch.bfloat16, device=x.device)
    F.call("glt_lm_head_fwd", _p(x), x.shape[0], D, _p(lm_head), _p(prepared), V, _p(out), _stream())
    return out


def lm_head_bwd(grad, lm_head, prepared=None):
    """dx [M,D] f32 = grad [M,V] . lm_head (the reference's grad_logits_full @
    lm_head, grafting.hip:1137)."""
    V, D = lm_head.shape
    if prepared is None:
        prepared = torch.empty(F.load().glt_lm_head_prepared_size(V, D), dtype=torch.uint8, device=grad.device)
        F.call("glt_lm_head_prepare", _p(lm_head), V, D, _p(prepared), _stream())
    dx = torch.empty((grad.shape[0], D), dtype=torch.float32, device=grad.device)
    F.call("glt_lm_head_bwd", _p(grad), grad.shape[0], V, _p(lm_head), _p(prepared), D, _p(dx), _stream())
    return dx


def embedding(ids, table):
    """table[ids] (at::embedding) for int32 ids, bf16 table [V,D]."""
    V, D = table.shape
    out = torch.empty((ids.numel(), D), dtype=torch.bfloat16, device=ids.device)
    F.call("glt_embedding", _p(ids), ids.numel(), _p(table), V, D, _p(out), _stream())
    return out


def eval_stats(logits, ids, hash_in=F.FNV_BASIS, reference_hash=True):
    """Shadow-eval terms of one batch (reference grafting.hip:504-547):
    dict(total_nll, count, ce, logits_sum, logits_sumsq, logits_hash).
    The hash is the reference's FNV-1a chain over every f32 logit byte,
    continued from hash_in (pass the previous batch's logits_hash to chain
    batches as the reference does); reference_hash=False gives the library's
    one-pass row form instead."""
    B, T = ids.shape
    V = logits.shape[-1]
    assert logits.stride(-1) == 1, "logits rows must be contiguous"
    ld = logits.stride(-2)
    lib = F.load()
    nbytes = lib.glt_eval_stats_workspace_size(B, T)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=logits.device)
    r = F.EvalResult()
    F.call("glt_eval_stats", _p(logits), ld, _p(ids), B, T, V,
           F.EVAL_HASH_REFERENCE if reference_hash else F.EVAL_HASH_ROWS, hash_in, ctypes.byref(r), _p(ws), nbytes,
           _stream())
    return {"total_nll": r.total_nll, "count": r.count, "ce": r.total_nll / max(r.count, 1),
            "logits_sum": r.logits_sum, "logits_sumsq": r.logits_sumsq, "logits_hash": r.logits_hash}


def eval_batches(batches, reference_hash=True):
    """The reference's whole eval loop over several (logits, ids) batches
    (grafting.hip:504-547): nll and counts summed, the logits hash chained
    from the FNV basis through every batch; returns the eval_stats dict of
    the whole set (ce = total_nll / count)."""
    out = {"total_nll": 0.0, "count": 0, "logits_sum": 0.0, "logits_sumsq": 0.0, "logits_hash": F.FNV_BASIS}
    for logits, ids in batches:
        r = eval_stats(logits, ids, out["logits_hash"], reference_hash)
        for k in ("total_nll", "count", "logits_sum", "logits_sumsq"):
            out[k] += r[k]
        out["logits_hash"] = r["logits_hash"]
    out["ce"] = out["total_nll"] / max(out["count"], 1)
    return out


def certify(A, B, C, D, ce_improve_margin=0.0, eps_ce_bake=0.02, eps_ce_reload=1e-4):
    """The A/B/C/D gates of the reference's certify step (deploy/certify.sh:28-59;
    default margins deploy/config.sh:39-41) over eval results (dicts with "ce"
    and "logits_hash"): A base, B explicit graft, C shadow-baked, D freshly
    reloaded base."""
    g1 = B["ce"] < A["ce"] - ce_improve_margin
    gap = C["ce"] - B["ce"]
    g2 = abs(gap) < eps_ce_bake
    g3 = abs(D["ce"] - A["ce"]) < eps_ce_reload and A["logits_hash"] == D["logits_hash"]
    content = "A_STANDALONE_DELTAS" if (g1 and g2) else ("B_BAKED_MISLABEL_SUSPECT" if g2 else "UNKNOWN")
    return {"A_ce": A["ce"], "B_ce": B["ce"], "C_ce": C["ce"], "D_ce": D["ce"], "A_hash": A["logits_hash"],
            "D_hash": D["logits_hash"], "gate_improve": int(g1), "gate_bake_equal": int(g2),
            "gate_reload_equal": int(g3), "bake_ce_gap": gap, "eps_ce_bake": eps_ce_bake, "content": content,
            "pass": int(g1 and g2 and g3)}

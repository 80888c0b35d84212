"""Python callables over the C-ABI, on torch device tensors (torch = device memory + streams only).

Names mirror the reference functions they replace:
  greedy_decode         <- EncoderDecoder.greedy_decode          (model.py:271-299)
  encode_latent         <- EncoderDecoder.get_latent / forward   (model.py:229-257)
  scorer_embed          <- SiameseNet.forward on like/unlike     (siamese_contrastive.py:381-382)
  scorer_edit_step      <- get_contrastive_loss + backward + Adam.step (:796-810)
  gemm_argmax           <- Generator + torch.max                 (model.py:200-207, :290-292)
  accept_changes        <- id2text_sentence compare + Change bookkeeping (:816-839)
Without a counterpart there: sample_logits / sample_decode (a draw in the argmax's place), quantize_weight_q4 / pack_weight_q4 /
gemm_q4 (products with 4-bit weights).
"""
import ctypes as C
import math

import torch

from . import _lib
from ._lib import check, lib


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


def _f32(t, shape=None):
    assert t.is_cuda and t.dtype == torch.float32 and t.is_contiguous(), "need contiguous f32 CUDA tensor"
    if shape is not None:
        assert tuple(t.shape) == tuple(shape), "shape %s != %s" % (tuple(t.shape), tuple(shape))
    return t


class DecodeWorkspace:
    """Grow-only device workspace shared by decode and encode calls."""

    def __init__(self, device):
        self.device = device
        self.buf = None

    def get(self, nbytes: int) -> torch.Tensor:
        if self.buf is None or self.buf.numel() < nbytes:
            self.buf = None
            self.buf = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        return self.buf


def decode_workspace_bytes(ae, B, max_len=60, l0_table=True):
    """device workspace st_decode_greedy needs for B decode jobs (K/V cache: 121 KB per job when the first layer reads
    the (token, position) table, 241 KB otherwise)"""
    return int(lib().st_decode_workspace_bytes_opt(C.byref(ae.dec), int(B), max_len, 0 if l0_table else _lib.ST_DEC_NO_L0_TABLE))


def greedy_decode(ae, latent, max_len=60, start_id=2, eos=3, pad=0, early_exit=True, sync_every=1,
                  want_gap=False, ws: DecodeWorkspace = None, screen=True, l0_table=True):
    """-> (ids [B,max_len-1] int32, gap or None, steps_run).
    screen=False (or want_gap=True) forces the full 3-product generator of the f16x3 format on every row."""
    _f32(latent)
    B = latent.shape[0]
    assert latent.shape[1] == 256
    T = max_len - 1
    ids = torch.empty(B, T, dtype=torch.int32, device=latent.device)
    gap = torch.empty(B, T, dtype=torch.float32, device=latent.device) if want_gap else None
    if B == 0:
        return ids, gap, 0
    options = ((_lib.ST_DEC_EARLY_EXIT if early_exit else 0) | (0 if screen else _lib.ST_DEC_NO_SCREEN) |
               (0 if l0_table else _lib.ST_DEC_NO_L0_TABLE))
    need = lib().st_decode_workspace_bytes_opt(C.byref(ae.dec), B, max_len, options)
    ws = ws or DecodeWorkspace(latent.device)
    buf = ws.get(need)
    steps = C.c_int(0)
    check(lib().st_decode_greedy(C.byref(ae.dec), latent.data_ptr(), B, max_len, start_id, eos, pad, options,
                                 sync_every, ids.data_ptr(), _p(gap),
                                 buf.data_ptr(), buf.numel(), C.byref(steps), _stream()), "st_decode_greedy")
    return ids, gap, steps.value


def encode_latent(ae, tokens, tok_pos, sent_off, n_sent, max_sent_len, ws: DecodeWorkspace = None, out=None):
    """Packed tokens (int32 device tensors) -> latent [n_sent,256] (written into `out`, a contiguous [n_sent,256] f32
    tensor, when given: the chunks of a large batch go straight into their rows of one buffer)."""
    R = tokens.numel()
    if out is not None:
        assert out.shape == (n_sent, 256) and out.dtype == torch.float32 and out.is_contiguous() and out.device == sent_off.device
    latent = out if out is not None else torch.empty(n_sent, 256, dtype=torch.float32, device=sent_off.device)
    if n_sent == 0:
        return latent
    need = lib().st_encode_workspace_bytes(C.byref(ae.enc), R, n_sent)
    ws = ws or DecodeWorkspace(latent.device)
    buf = ws.get(max(need, 256))
    check(lib().st_encode_latent(C.byref(ae.enc), _p(tokens), _p(tok_pos), sent_off.data_ptr(), R, n_sent,
                                 max_sent_len, latent.data_ptr(), buf.data_ptr(), buf.numel(), _stream()),
          "st_encode_latent")
    return latent


def scorer_embed(sw, x, unit=True):
    _f32(x)
    n = x.shape[0]
    z = torch.empty_like(x)
    check(lib().st_scorer_embed(C.byref(sw.c), x.data_ptr(), z.data_ptr(), n, 1 if unit else 0, _stream()),
          "st_scorer_embed")
    return z


def scorer_edit_step(sw, latent, adam_m, adam_v, like_z, unlike_z, lr, step, active, tau=0.1, not_nll=False,
                     simplest=False, just_use_one=False, want_loss=False, want_grad=False, want_scores=False, optimizer="Adam"):
    """-> (loss, grad), or (loss, grad, scores [B, n_pos + n_neg]) with want_scores.
    optimizer: a torch.optim name (siamese_contrastive.py:780) out of _lib.ST_OPTIMIZERS; adam_m / adam_v are its state."""
    if optimizer not in _lib.ST_OPTIMIZERS:
        raise NotImplementedError("--victim_optimizer %s: the kernel has %s" % (optimizer, ", ".join(_lib.ST_OPTIMIZERS)))
    B = latent.shape[0]
    _f32(latent, (B, 256)); _f32(adam_m, (B, 256)); _f32(adam_v, (B, 256)); _f32(lr, (B,))
    n_pos = 0 if like_z is None else like_z.shape[1]
    n_neg = 0 if unlike_z is None else unlike_z.shape[1]
    if like_z is not None:
        _f32(like_z, (B, n_pos, 256))
    if unlike_z is not None:
        _f32(unlike_z, (B, n_neg, 256))
    assert step.dtype == torch.int32 and step.is_cuda
    assert active is None or (active.dtype == torch.uint8 and active.is_cuda)
    flags = (_lib.ST_F_NOT_NLL if not_nll else 0) | (_lib.ST_F_SIMPLEST if simplest else 0) | \
            (_lib.ST_F_JUST_USE_ONE if just_use_one else 0) | (_lib.ST_OPTIMIZERS[optimizer] << _lib.ST_F_OPT_SHIFT)
    loss = torch.empty(B, dtype=torch.float32, device=latent.device) if want_loss else None
    grad = torch.empty(B, 256, dtype=torch.float32, device=latent.device) if want_grad else None
    scores = torch.empty(B, n_pos + n_neg, dtype=torch.float32, device=latent.device) if want_scores else None
    check(lib().st_scorer_edit_step(C.byref(sw.c), latent.data_ptr(), adam_m.data_ptr(), adam_v.data_ptr(),
                                    _p(like_z), _p(unlike_z), n_pos, n_neg, lr.data_ptr(), step.data_ptr(),
                                    _p(active), B, float(tau), flags, _p(loss), _p(grad), _p(scores), _stream()),
          "st_scorer_edit_step")
    return (loss, grad, scores) if want_scores else (loss, grad)


def _fmt(gemm_format):
    if isinstance(gemm_format, str):
        if gemm_format not in _lib.GEMM_FORMATS:
            raise ValueError("gemm_format %r: expected one of %s" % (gemm_format, sorted(_lib.GEMM_FORMATS)))
        return _lib.GEMM_FORMATS[gemm_format]
    return int(gemm_format)


def pack_weight(W, gemm_format="f32"):
    """nn.Linear weight [N,K] (device f32) -> MFMA-fragment-ordered image (st_pack_weight) for the
    exact f32 kernels ("f32") or the 3-product f16 split kernels ("f16x3")."""
    _f32(W)
    N, K = W.shape
    out = torch.empty(lib().st_packed_weight_floats(N, K), dtype=torch.float32, device=W.device)
    check(lib().st_pack_weight(W.data_ptr(), N, K, _fmt(gemm_format), out.data_ptr(), _stream()), "st_pack_weight")
    return out


def gemm_argmax(h, W, b, ln_a=None, ln_b=None, packed=None, gemm_format="f32"):
    """W [V,256] plain (packed here) or pass packed=pack_weight(W, gemm_format)."""
    _f32(h); _f32(b)
    n, V = h.shape[0], b.shape[0]
    assert h.shape[1] == 256
    W = packed if packed is not None else pack_weight(W, gemm_format)
    ids = torch.empty(n, dtype=torch.int32, device=h.device)
    best = torch.empty(n, dtype=torch.float32, device=h.device)
    gap = torch.empty(n, dtype=torch.float32, device=h.device)
    scratch = torch.empty(max(n, 1) * _lib.ST_ARGMAX_SPLITS * 16, dtype=torch.uint8, device=h.device)
    check(lib().st_gemm_argmax(h.data_ptr(), _p(ln_a), _p(ln_b), W.data_ptr(), b.data_ptr(), n, V, _fmt(gemm_format),
                               ids.data_ptr(), best.data_ptr(), gap.data_ptr(), scratch.data_ptr(), _stream()), "st_gemm_argmax")
    return ids, best, gap


def gemm_argmax_noalloc(h, packed, b, ids, best, gap, ln_a=None, ln_b=None, gemm_format="f32"):
    """st_gemm_argmax_noalloc: every buffer (inputs AND outputs) comes from the caller, the scratch is the library's
    static device array; this wrapper allocates nothing either.  n <= _lib.ST_NOALLOC_MAX_ROWS."""
    _f32(h); _f32(b); _f32(best); _f32(gap)
    n, V = h.shape[0], b.shape[0]
    assert h.shape[1] == 256 and ids.dtype == torch.int32 and ids.numel() >= n and best.numel() >= n and gap.numel() >= n
    check(lib().st_gemm_argmax_noalloc(h.data_ptr(), _p(ln_a), _p(ln_b), packed.data_ptr(), b.data_ptr(), n, V,
                                       _fmt(gemm_format), ids.data_ptr(), best.data_ptr(), gap.data_ptr(), _stream()),
          "st_gemm_argmax_noalloc")


def accept_changes(new_ids, acc_ids, vocab, n_changes, changed, active, max_change=7, unk=1, eos=3, pad=0,
                   canon=None, rec_ids=None, confirm_ids=None):
    B, T = new_ids.shape
    assert new_ids.dtype == torch.int32 and acc_ids.dtype == torch.int32 and new_ids.is_contiguous() and acc_ids.is_contiguous()
    check(lib().st_accept_changes(new_ids.data_ptr(), acc_ids.data_ptr(), T, B, vocab, unk, eos, pad, _p(canon),
                                  max_change, n_changes.data_ptr(), changed.data_ptr(), active.data_ptr(),
                                  _p(rec_ids), _p(confirm_ids), _stream()), "st_accept_changes")


def simloss_format(gemm_format):
    """operand format of the similarity products ("f16x3" default, "f32" exact); returns the previous one"""
    prev = lib().st_simloss_format(_fmt(gemm_format))
    return {v: k for k, v in _lib.GEMM_FORMATS.items()}[prev]


def simloss_fwd(ori, like, tau=0.1, row_offset=0):
    """-> (loss [Bq], lse [Bq]) of the in-batch InfoNCE block (siamese_contrastive.py:1060-1069)."""
    _f32(ori); _f32(like)
    Bq, Bk = ori.shape[0], like.shape[0]
    loss = torch.empty(Bq, dtype=torch.float32, device=ori.device)
    lse = torch.empty(Bq, dtype=torch.float32, device=ori.device)
    nb = lib().st_simloss_scratch_bytes(Bq, Bk)
    scratch = torch.empty(nb, dtype=torch.uint8, device=ori.device)
    check(lib().st_simloss_fwd(ori.data_ptr(), like.data_ptr(), Bq, Bk, float(tau), row_offset, loss.data_ptr(),
                               lse.data_ptr(), scratch.data_ptr(), nb, _stream()), "st_simloss_fwd")
    return loss, lse


def simloss_bwd(ori, like, lse, g, tau=0.1, row_offset=0, d_like=None):
    """-> (d_ori [Bq,256], d_like [Bk,256]); d_like is accumulated into when given."""
    Bq, Bk = ori.shape[0], like.shape[0]
    d_ori = torch.empty_like(ori)
    if d_like is None:
        d_like = torch.zeros_like(like)
    nb = lib().st_simloss_scratch_bytes(Bq, Bk)
    scratch = torch.empty(nb, dtype=torch.uint8, device=ori.device)
    check(lib().st_simloss_bwd(ori.data_ptr(), like.data_ptr(), Bq, Bk, float(tau), row_offset, lse.data_ptr(),
                               g.data_ptr(), d_ori.data_ptr(), d_like.data_ptr(), scratch.data_ptr(), nb, _stream()),
          "st_simloss_bwd")
    return d_ori, d_like


def fgim_perturb(cw, latent, target, eps, want_grad=False):
    """Classifier forward + BCE backward to the latent + x - eps_k * grad (fgim_attack, model.py:454-516).
    latent [B,256], target [B] (0/1), eps: sequence of step sizes -> (pred [B], grad [B,256] or None, out [n_eps,B,256])."""
    _f32(latent)
    B = latent.shape[0]
    target = target.to(device=latent.device, dtype=torch.float32).contiguous().view(-1)
    assert target.numel() == B and latent.shape[1] == 256
    e = torch.as_tensor(list(eps), dtype=torch.float32, device=latent.device)
    pred = torch.empty(B, dtype=torch.float32, device=latent.device)
    grad = torch.empty(B, 256, dtype=torch.float32, device=latent.device) if want_grad else None
    out = torch.empty(e.numel(), B, 256, dtype=torch.float32, device=latent.device)
    check(lib().st_fgim_perturb(C.byref(cw.c), latent.data_ptr(), target.data_ptr(), e.data_ptr(), e.numel(), B,
                                pred.data_ptr(), _p(grad), out.data_ptr(), _stream()), "st_fgim_perturb")
    return pred, grad, out


# ---- products with 4-bit weights, and a draw from the logits (no counterpart in the reference) -----------------------

_TYPES = {torch.float32: _lib.ST_TYPE_F32, torch.bfloat16: _lib.ST_TYPE_BF16, torch.float16: _lib.ST_TYPE_F16}


def _on(t, name, dtype, shape, device=None):
    """a contiguous GPU tensor of this type and shape, or a ValueError that names it"""
    if not (torch.is_tensor(t) and t.is_cuda and t.dtype == dtype and tuple(t.shape) == tuple(shape) and t.is_contiguous()):
        raise ValueError("%s: expected a contiguous %s GPU tensor of shape %s, got %s" % (
            name, dtype, tuple(shape), "%s %s on %s" % (t.dtype, tuple(t.shape), t.device) if torch.is_tensor(t) else type(t).__name__))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    return t


def _rows_of(t, name):
    """-> (type, values between rows) of a 2-d GPU tensor whose rows are contiguous"""
    if not (torch.is_tensor(t) and t.is_cuda and t.dim() == 2 and t.dtype in _TYPES):
        raise ValueError("%s: expected a 2-d float32, bfloat16 or float16 GPU tensor" % name)
    ld, one = t.stride()
    if one != 1 and t.shape[1] > 1:
        raise ValueError("%s: the values of a row must be contiguous (stride %s)" % (name, t.stride()))
    return _TYPES[t.dtype], ld


def _call(device, name, *args):
    """one call of the library on `device`'s current stream, whichever device is current.  (The stream's bare handle: a Stream
    object around it costs 2.7 us of a 7 us call.)"""
    fn, i = getattr(lib(), name), device.index
    if i == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc != 0:
        check(rc, name)


def _q4_sides(N, K):
    """sizes that the library takes (and that its 32-bit arguments hold)"""
    if max(N, K) > _lib.ST_Q4_MAX_SIDE:
        raise ValueError("a [%d, %d] weight: at most %d rows and columns" % (N, K, _lib.ST_Q4_MAX_SIDE))


class Q4Weight:
    """A packed [N, K] weight of 4-bit codes with a scale (and a zero code) per group of columns: st_pack_weight_q4's image
    and the struct that st_gemm_q4 takes."""

    def __init__(self, image, N, K, group, has_zeros):
        self.image, self.N, self.K, self.group = image, N, K, group
        self.c = _lib.StQ4Weight(image.data_ptr(), N, K, group, 1 if has_zeros else 0)
        self.ref = C.byref(self.c)


def quantize_weight_q4(W, group=128, zero_points=False):
    """nn.Linear weight [N, K] (f32) -> (codes u8 [N, ceil(K/2)], scales f16 [N, ceil(K/group)], zeros u8 or None):
    scale = max |w| / 7 of the group, with zero_points (max - min) / 15; W ~ scale * (code - zero), zero = 8 when None."""
    if not (torch.is_tensor(W) and W.is_cuda and W.dim() == 2 and W.dtype == torch.float32 and W.is_contiguous() and W.numel()):
        raise ValueError("W: expected a contiguous 2-d float32 GPU tensor")
    if group not in (32, 64, 128):
        raise ValueError("group %r: expected 32, 64 or 128" % (group,))
    N, K = W.shape
    _q4_sides(N, K)
    g = -(-K // group)
    codes = torch.empty(N, (K + 1) // 2, dtype=torch.uint8, device=W.device)
    scales = torch.empty(N, g, dtype=torch.float16, device=W.device)
    zeros = torch.empty(N, g, dtype=torch.uint8, device=W.device) if zero_points else None
    _call(W.device, "st_quantize_weight_q4", W.data_ptr(), N, K, group, codes.data_ptr(), scales.data_ptr(), _p(zeros))
    return codes, scales, zeros


def pack_weight_q4(codes, scales, zeros=None, k=None, group=128):
    """4-bit codes (two a byte, even columns low), f16 group scales and zero codes of a [N, k] weight -> Q4Weight
    (st_pack_weight_q4).  k defaults to twice the bytes of a row (give it where it is odd)."""
    if not (torch.is_tensor(codes) and codes.is_cuda and codes.dim() == 2 and codes.dtype == torch.uint8 and codes.is_contiguous()):
        raise ValueError("codes: expected a contiguous 2-d uint8 GPU tensor")
    if group not in (32, 64, 128):
        raise ValueError("group %r: expected 32, 64 or 128" % (group,))
    N = codes.shape[0]
    K = 2 * codes.shape[1] if k is None else int(k)
    if K < 1 or (K + 1) // 2 != codes.shape[1]:
        raise ValueError("codes: %d bytes a row do not hold k = %d columns" % (codes.shape[1], K))
    _q4_sides(N, K)
    shape = (N, -(-K // group))
    _on(scales, "scales", torch.float16, shape, codes.device)
    if zeros is not None:
        _on(zeros, "zeros", torch.uint8, shape, codes.device)
    nbytes = lib().st_q4_packed_bytes(N, K, group, 0 if zeros is None else 1)
    image = torch.empty(nbytes, dtype=torch.uint8, device=codes.device)
    _call(codes.device, "st_pack_weight_q4", codes.data_ptr(), scales.data_ptr(), _p(zeros), N, K, group, image.data_ptr())
    return Q4Weight(image, N, K, group, zeros is not None)


def _share_values(a, b):
    """whether two 2-d tensors, the values of a row contiguous, have a byte in common; columns of one buffer, side by side, have none"""
    if 0 in a.shape or 0 in b.shape:
        return False
    p, q, wide_a, wide_b = a.data_ptr(), b.data_ptr(), a.shape[1] * a.element_size(), b.shape[1] * b.element_size()
    row, row_b = a.stride(0) * a.element_size(), b.stride(0) * b.element_size()
    if p + (a.shape[0] - 1) * row + wide_a <= q or q + (b.shape[0] - 1) * row_b + wide_b <= p:
        return False
    if b.shape[0] == 1:
        row_b = row
    if row != row_b or row == 0:
        return True
    off = (q - p) % row
    return not (off >= wide_a and off + wide_b <= row)


def gemm_q4(x, weight, bias=None, out=None):
    """x [M, K] (f32, bf16 or f16; rows may be strided) times a Q4Weight's transpose, plus bias f32 [N] -> [M, N] of x's type
    (written into `out` when given: same type, rows may be strided, no value of x's or the bias's).  Has no gradient: where one
    would be lost (grad mode on, x or bias requires it) the call is refused."""
    kind, ldx = _rows_of(x, "x")
    M, dev = x.shape[0], x.device
    if M > _lib.ST_Q4_MAX_ROWS:
        raise ValueError("x has %d rows: at most %d in one call" % (M, _lib.ST_Q4_MAX_ROWS))
    if x.shape[1] != weight.K:
        raise ValueError("x has %d columns, the weight %d" % (x.shape[1], weight.K))
    if weight.image.device != dev:
        raise ValueError("the weight is on %s, x on %s" % (weight.image.device, dev))
    if bias is not None:
        _on(bias, "bias", torch.float32, (weight.N,), dev)
    if (x.requires_grad or (bias is not None and bias.requires_grad)) and torch.is_grad_enabled():
        raise ValueError("gemm_q4 has no gradient: call it under torch.no_grad(), or with detached tensors")
    if out is None:
        out, ldy = torch.empty(M, weight.N, dtype=x.dtype, device=dev), weight.N
    else:
        ldy = _rows_of(out, "out")[1]
        if out.dtype != x.dtype or tuple(out.shape) != (M, weight.N) or out.device != dev:
            raise ValueError("out: expected %s of shape %s on %s" % (x.dtype, (M, weight.N), dev))
        if _share_values(x, out):
            raise ValueError("out shares values with x")
        if bias is not None and _share_values(out, bias[None]):
            raise ValueError("out shares values with bias")
    _call(dev, "st_gemm_q4", x.data_ptr(), kind, ldx, M, weight.ref, _p(bias), out.data_ptr(), ldy)
    return out


def _sample_settings(B, dev, temperature, top_k, top_p, min_p):
    """-> (StSampleSettings, what it points to); a setting is a number, or a tensor [B] (f32, top_k int32) on the GPU"""
    s = _lib.StSampleSettings(1.0, 0, 1.0, 0.0)
    if torch.is_tensor(temperature):
        s.temperature_rows = _on(temperature, "temperature", torch.float32, (B,), dev).data_ptr()
    elif 0.0 <= temperature < math.inf:
        s.temperature = temperature
    else:
        raise ValueError("temperature %r: expected a finite number of at least 0" % (temperature,))
    if torch.is_tensor(top_k):
        s.top_k_rows = _on(top_k, "top_k", torch.int32, (B,), dev).data_ptr()
    elif int(top_k) == top_k and 0 <= top_k < 1 << 31:
        s.top_k = int(top_k)
    else:
        raise ValueError("top_k %r: expected a whole number, 0 for off" % (top_k,))
    if torch.is_tensor(top_p):
        s.top_p_rows = _on(top_p, "top_p", torch.float32, (B,), dev).data_ptr()
    elif 0.0 < top_p <= 1.0:
        s.top_p = top_p
    else:
        raise ValueError("top_p %r: expected a number in (0, 1]" % (top_p,))
    if torch.is_tensor(min_p):
        s.min_p_rows = _on(min_p, "min_p", torch.float32, (B,), dev).data_ptr()
    elif 0.0 <= min_p <= 1.0:
        s.min_p = min_p
    else:
        raise ValueError("min_p %r: expected a number in [0, 1]" % (min_p,))
    return s


def _workspace(ws, nbytes, device):
    """a DecodeWorkspace's buffer, or one for this call alone.  A graph that is being captured gets one from its own pool: the
    DecodeWorkspace's may be replaced by a larger one, or serve another graph, before the replay."""
    if ws is None or torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    buf = ws.get(nbytes)
    if buf.device != device:
        raise ValueError("ws is on %s, not on %s" % (buf.device, device))
    buf.record_stream(torch.cuda.current_stream(device))   # a larger one may replace it while this call still runs
    return buf


def sample_logits(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, want_logp=True, ws: DecodeWorkspace = None):
    """One token per row of logits [B, V] (f32, bf16 or f16; rows may be strided) from the uniform numbers u [B] (f32, in
    [0, 1)) -> (ids int32 [B], logp f32 [B] or None).  Filters in the order temperature, top_k (0: off), top_p (1: off),
    min_p (0: off); each is a number or a tensor [B].  temperature 0: argmax.  A row of -inf / NaN alone: id -1, logp -inf.
    logp is a value: no gradient goes from it to the logits.  Calls that may run at the same time need a ws each, or none."""
    kind, ld = _rows_of(logits, "logits")
    B, V = logits.shape
    dev = logits.device
    if V < 1 or V > _lib.ST_SAMPLE_MAX_VOCAB:
        raise ValueError("logits: rows of %d values (1 .. %d)" % (V, _lib.ST_SAMPLE_MAX_VOCAB))
    if B >= 1 << 31:
        raise ValueError("logits: %d rows do not fit into 32 bits" % B)
    _on(u, "u", torch.float32, (B,), dev)
    s = _sample_settings(B, dev, temperature, top_k, top_p, min_p)
    ids = torch.empty(B, dtype=torch.int32, device=dev)
    logp = torch.empty(B, dtype=torch.float32, device=dev) if want_logp else None
    nbytes = lib().st_sample_workspace_bytes(B, V)
    buf = None if nbytes == 0 else _workspace(ws, nbytes, dev)
    _call(dev, "st_sample_logits", logits.data_ptr(), kind, ld, B, V, u.data_ptr(), C.byref(s), ids.data_ptr(), _p(logp), _p(buf), nbytes)
    return ids, logp


def sample_decode(ae, latent, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, head=None, max_len=60, start_id=2, eos=3, pad=0,
                  early_exit=True, sync_every=1, want_logp=True, ws: DecodeWorkspace = None, l0_table=True):
    """greedy_decode with a draw in the argmax's place (st_decode_sample): latent [B, 256], uniform numbers u [B, max_len - 1]
    (f32, in [0, 1)) -> (ids int32 [B, max_len - 1], logp f32 of the same shape or None, steps run).  Settings as sample_logits,
    numbers or tensors [B].  head: the generator as a Q4Weight (ae.quantized_generator()), None: as the weights were packed.  The
    4-bit head makes a step of up to some 256 sentences shorter, of many it does not (1: 146 -> 130 us, 4096: 377 -> 412 us); its
    products are split-f16 ones (st_gemm_q4's error) whatever the weights' gemm_format.  temperature 0 gives greedy_decode's tokens."""
    if not (torch.is_tensor(latent) and latent.dim() == 2 and latent.shape[1] == 256):
        raise ValueError("latent: expected [B, 256]")
    B, T, dev = latent.shape[0], max_len - 1, latent.device
    _on(latent, "latent", torch.float32, (B, 256))
    if ae.where != dev:
        raise ValueError("the weights are on %s, latent on %s" % (ae.where, dev))
    _on(u, "u", torch.float32, (B, T), dev)
    if head is not None and (not isinstance(head, Q4Weight) or (head.N, head.K) != (ae.vocab, 256) or head.image.device != dev):
        raise ValueError("head: expected a Q4Weight [%d, 256] on %s" % (ae.vocab, dev))
    s = _sample_settings(B, dev, temperature, top_k, top_p, min_p)
    ids = torch.empty(B, T, dtype=torch.int32, device=dev)
    logp = torch.empty(B, T, dtype=torch.float32, device=dev) if want_logp else None
    if B == 0:
        return ids, logp, 0
    options = (_lib.ST_DEC_EARLY_EXIT if early_exit else 0) | (0 if l0_table else _lib.ST_DEC_NO_L0_TABLE)
    need = lib().st_decode_sample_workspace_bytes(C.byref(ae.dec), B, max_len, options)
    buf = _workspace(ws, need, dev)
    steps = C.c_int(0)
    _call(dev, "st_decode_sample", C.byref(ae.dec), None if head is None else head.ref, latent.data_ptr(), B, max_len, start_id, eos, pad,
          options, sync_every, u.data_ptr(), C.byref(s), ids.data_ptr(), _p(logp), buf.data_ptr(), buf.numel(), C.byref(steps))
    return ids, logp, steps.value

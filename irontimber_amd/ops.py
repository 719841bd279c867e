"""Torch-tensor front end over the C ABI (device memory and streams come from PyTorch-ROCm).

Each function validates dtypes/devices/contiguity, then calls the matching `it_*` entry point on
torch's current stream. Buffer layouts and semantics are those of include/it_attn.h.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from ._lib import ItError, Kv8CacheArgs, call, last_error, lib

KERNEL_AUTO, KERNEL_SPLITK, KERNEL_FLASH, KERNEL_FLASH_F32 = 0, 1, 2, 3


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _need(t: torch.Tensor, dtype: torch.dtype, name: str):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def kv_append_f16(k: torch.Tensor, v: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int,
                  round_mode: int = 0) -> None:
    """Append k, v [nt, kvd] f32 to the f16 caches kc, vc [ctx, kvd] (stored as int16 bits or f16)."""
    _need(k, torch.float32, "k"); _need(v, torch.float32, "v")
    nt, kvd = k.shape
    for c in (kc, vc):
        if c.dtype not in (torch.float16, torch.int16) or not c.is_contiguous() or c.shape[-1] != kvd:
            raise ValueError("kc/vc must be contiguous [ctx, kvd] f16")
        if c.shape[0] < pos0 + nt:
            raise ValueError("cache too short")
    call("it_kv_append_f16", k.data_ptr(), v.data_ptr(), kvd, kc.data_ptr(), vc.data_ptr(), pos0, nt, kvd,
         round_mode, _stream())


def attn_prep_f16(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int,
                  nh: int, nkv: int, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                  eps: float = 1e-6, n_rot: int = 64, theta_scale: float | None = None, rope_base: float = 1e7,
                  sections=(11, 11, 10, 0), round_mode: int = 0) -> None:
    """Norm + rope of q (in place, q [nt, nh*2*hd]) and k [nt, nkv*hd], then the f16 append of k and
    v to kc/vc at rows pos0.. (it_attn_prep_f16). theta_scale defaults to rope_base^(-2/n_rot) in f32."""
    _need(q, torch.float32, "q"); _need(k, torch.float32, "k"); _need(v, torch.float32, "v")
    nt, kvd = k.shape
    hd = kvd // nkv
    if q.shape != (nt, nh * 2 * hd) or v.shape != k.shape:
        raise ValueError("q must be [nt, nh*2*hd] and v the shape of k [nt, nkv*hd]")
    for c in (kc, vc):
        if c.dtype not in (torch.float16, torch.int16) or not c.is_contiguous() or c.shape[-1] != kvd:
            raise ValueError("kc/vc must be contiguous [ctx, kvd] f16")
        if c.shape[0] < pos0 + nt:
            raise ValueError("cache too short")
    for w, n in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if w is not None:
            _need(w, torch.float32, n)
            if w.numel() != hd:
                raise ValueError(f"{n} must hold head_dim floats")
    if theta_scale is None:
        from .synth import rope_theta_scale
        theta_scale = rope_theta_scale(rope_base, n_rot)
    s = list(sections) + [0] * (4 - len(sections))
    call("it_attn_prep_f16", q.data_ptr(), q.shape[1], k.data_ptr(), v.data_ptr(), kvd, _ptr(q_norm), _ptr(k_norm),
         float(eps), kc.data_ptr(), vc.data_ptr(), kvd, pos0, hd, nh, nkv, nt, n_rot, float(theta_scale), *s[:4],
         round_mode, _stream())


def attn_prep_f16_q16(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int,
                      nh: int, nkv: int, scale: float | None = None, q_norm: torch.Tensor | None = None,
                      k_norm: torch.Tensor | None = None, eps: float = 1e-6, n_rot: int = 64,
                      theta_scale: float | None = None, rope_base: float = 1e7, sections=(11, 11, 10, 0),
                      round_mode: int = 0) -> torch.Tensor:
    """attn_prep_f16 that also returns q16 [nt, nh*hd] f16 = f16(q' * scale * log2(e)), the flash
    prefill kernel's query operand for attn_f16_q16 with the same scale (it_attn_prep_f16_q16)."""
    _need(q, torch.float32, "q"); _need(k, torch.float32, "k"); _need(v, torch.float32, "v")
    nt, kvd = k.shape
    hd = kvd // nkv
    if q.shape != (nt, nh * 2 * hd) or v.shape != k.shape:
        raise ValueError("q must be [nt, nh*2*hd] and v the shape of k [nt, nkv*hd]")
    for c in (kc, vc):
        if c.dtype not in (torch.float16, torch.int16) or not c.is_contiguous() or c.shape[-1] != kvd:
            raise ValueError("kc/vc must be contiguous [ctx, kvd] f16")
        if c.shape[0] < pos0 + nt:
            raise ValueError("cache too short")
    if scale is None:
        scale = 1.0 / hd ** 0.5
    if theta_scale is None:
        from .synth import rope_theta_scale
        theta_scale = rope_theta_scale(rope_base, n_rot)
    q16 = torch.empty(nt, nh * hd, device=q.device, dtype=torch.float16)
    s = list(sections) + [0] * (4 - len(sections))
    call("it_attn_prep_f16_q16", q.data_ptr(), q.shape[1], k.data_ptr(), v.data_ptr(), kvd, _ptr(q_norm),
         _ptr(k_norm), float(eps), kc.data_ptr(), vc.data_ptr(), kvd, pos0, hd, nh, nkv, nt, n_rot, float(theta_scale),
         *s[:4], round_mode, q16.data_ptr(), nh * hd, float(scale), _stream())
    return q16


def attn_prep_f32kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int,
                    row0: int, nh: int, nkv: int, q_norm: torch.Tensor | None = None,
                    k_norm: torch.Tensor | None = None, eps: float = 1e-6, n_rot: int = 64,
                    theta_scale: float | None = None, rope_base: float = 1e7, sections=(11, 11, 10, 0)) -> None:
    """attn_prep_f16 for an f32 cache: rope at positions pos0.., K/V rows stored at cache rows row0..
    (the MTP head stores position p in row p - 1)."""
    _need(q, torch.float32, "q"); _need(k, torch.float32, "k"); _need(v, torch.float32, "v")
    _need(kc, torch.float32, "kc"); _need(vc, torch.float32, "vc")
    nt, kvd = k.shape
    hd = kvd // nkv
    if q.shape != (nt, nh * 2 * hd) or v.shape != k.shape:
        raise ValueError("q must be [nt, nh*2*hd] and v the shape of k [nt, nkv*hd]")
    for c in (kc, vc):
        if c.shape[-1] != kvd or c.shape[0] < row0 + nt:
            raise ValueError("kc/vc must be [rows >= row0 + nt, kvd] f32")
    if theta_scale is None:
        from .synth import rope_theta_scale
        theta_scale = rope_theta_scale(rope_base, n_rot)
    s = list(sections) + [0] * (4 - len(sections))
    call("it_attn_prep_f32kv", q.data_ptr(), q.shape[1], k.data_ptr(), v.data_ptr(), kvd, _ptr(q_norm), _ptr(k_norm),
         float(eps), kc.data_ptr(), vc.data_ptr(), kvd, pos0, row0, hd, nh, nkv, nt, n_rot, float(theta_scale), *s[:4],
         _stream())


def attn_f32kv(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int, nh: int, nkv: int,
               scale: float | None = None, out: torch.Tensor | None = None,
               scratch: torch.Tensor | None = None) -> torch.Tensor:
    """q [nt, nh*2*hd] f32 (q | gate per head), kc/vc [rows, nkv*hd] f32 -> out [nt, nh*hd] f32;
    query t sees rows 0..pos0+t."""
    _need(q, torch.float32, "q"); _need(kc, torch.float32, "kc"); _need(vc, torch.float32, "vc")
    nt = q.shape[0]
    hd = q.shape[-1] // (2 * nh)
    kvd = nkv * hd
    for c in (kc, vc):
        if c.shape[-1] != kvd or c.shape[0] < pos0 + nt:
            raise ValueError("kc/vc must be [rows >= pos0 + nt, nkv*hd] f32")
    if scale is None:
        scale = 1.0 / hd ** 0.5
    if out is None:
        out = torch.empty(nt, nh * hd, device=q.device, dtype=torch.float32)
    if scratch is None:
        need = lib().it_attn_f32kv_scratch_bytes(pos0, nt, hd, nh, nkv)
        scratch = torch.empty(max(need, 16), device=q.device, dtype=torch.uint8)
    sp, sb = (scratch.data_ptr(), scratch.numel() * scratch.element_size()) if scratch.numel() else (None, 0)
    call("it_attn_f32kv", q.data_ptr(), nh * 2 * hd, kc.data_ptr(), vc.data_ptr(), kvd, pos0, hd, nh, nkv, nt,
         float(scale), out.data_ptr(), nh * hd, sp, sb, _stream())
    return out


def attn_scratch_bytes(pos0: int, nt: int, nh: int, nkv: int, hd: int = 256, kernel: int = KERNEL_AUTO,
                       chunk: int = 0) -> int:
    return lib().it_attn_scratch_bytes_ex(pos0, nt, hd, nh, nkv, kernel, chunk)


def attn_f16(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int, nh: int, nkv: int,
             scale: float | None = None, out: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
             kernel: int = KERNEL_AUTO, chunk: int = 0) -> torch.Tensor:
    """q [nt, nh*2*hd] f32 (q | gate per head), kc/vc [ctx, nkv*hd] f16 -> out [nt, nh*hd] f32."""
    _need(q, torch.float32, "q")
    nt = q.shape[0]
    hd = q.shape[-1] // (2 * nh) if q.dim() == 2 else q.shape[-1] // 2
    kvd = nkv * hd
    if scale is None:
        scale = 1.0 / hd ** 0.5
    for c in (kc, vc):
        if c.dtype not in (torch.float16, torch.int16) or not c.is_contiguous() or c.shape[-1] != kvd:
            raise ValueError("kc/vc must be contiguous [ctx, nkv*hd] f16")
        if c.shape[0] < pos0 + nt:
            raise ValueError("cache shorter than pos0 + nt")
    if out is None:
        out = torch.empty(nt, nh * hd, device=q.device, dtype=torch.float32)
    _need(out, torch.float32, "out")
    need = attn_scratch_bytes(pos0, nt, nh, nkv, hd, kernel, chunk)
    if scratch is None and need:
        scratch = torch.empty(need, device=q.device, dtype=torch.uint8)
    nbytes = 0 if scratch is None else scratch.numel() * scratch.element_size()
    call("it_attn_f16_ex", q.data_ptr(), nh * 2 * hd, kc.data_ptr(), vc.data_ptr(), kvd, pos0, hd, nh, nkv, nt,
         float(scale), out.data_ptr(), nh * hd, _ptr(scratch), nbytes, kernel, chunk, _stream())
    return out


def attn_f16_q16(q: torch.Tensor, q16: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int, nh: int, nkv: int,
                 scale: float | None = None, out: torch.Tensor | None = None,
                 scratch: torch.Tensor | None = None) -> torch.Tensor:
    """attn_f16 with the flash kernel's query operand given as q16 [nt, nh*hd] f16 (attn_prep_f16_q16
    with the same scale, or f16(q * scale * log2(e))); q still gives the gates (it_attn_f16_q16)."""
    _need(q, torch.float32, "q")
    nt = q.shape[0]
    hd = q.shape[-1] // (2 * nh)
    kvd = nkv * hd
    if scale is None:
        scale = 1.0 / hd ** 0.5
    if q16.dtype != torch.float16 or not q16.is_contiguous() or q16.shape != (nt, nh * hd):
        raise ValueError("q16 must be contiguous [nt, nh*hd] f16")
    for c in (kc, vc):
        if c.dtype not in (torch.float16, torch.int16) or not c.is_contiguous() or c.shape[-1] != kvd:
            raise ValueError("kc/vc must be contiguous [ctx, nkv*hd] f16")
        if c.shape[0] < pos0 + nt:
            raise ValueError("cache shorter than pos0 + nt")
    if out is None:
        out = torch.empty(nt, nh * hd, device=q.device, dtype=torch.float32)
    _need(out, torch.float32, "out")
    if scratch is None:
        need = attn_scratch_bytes(pos0, nt, nh, nkv, hd)
        scratch = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
    nbytes = 0 if scratch is None else scratch.numel() * scratch.element_size()
    call("it_attn_f16_q16", q.data_ptr(), nh * 2 * hd, q16.data_ptr(), nh * hd, kc.data_ptr(), vc.data_ptr(), kvd,
         pos0, hd, nh, nkv, nt, float(scale), out.data_ptr(), nh * hd, _ptr(scratch), nbytes, _stream())
    return out


def attn_mailbox(ctx: int, nt: int, nh: int, device) -> torch.Tensor:
    """A mailbox for attn_f16_mailbox (decode / verify rows up to nt at context up to ctx, nh
    heads), initialised on the current stream. Keep one per stream of calls."""
    nbytes = lib().it_attn_mailbox_bytes(ctx, nt, nh)
    mb = torch.empty(nbytes, device=device, dtype=torch.uint8)
    call("it_attn_mailbox_init", mb.data_ptr(), nbytes, _stream())
    return mb


def attn_mailbox_poisoned(mb: torch.Tensor) -> bool:
    """True if a one-launch merge in this mailbox ever gave up waiting (synchronises the stream)."""
    flag = ctypes.c_int(0)
    call("it_attn_mailbox_poisoned", mb.data_ptr(), ctypes.addressof(flag), _stream())
    return bool(flag.value)


def attn_mailbox_would_launch(pos0: int, nt: int, nh: int, nkv: int, mailbox: torch.Tensor, hd: int = 256) -> bool:
    """Whether attn_f16_mailbox takes the one-launch form for this geometry and mailbox."""
    return bool(lib().it_attn_mailbox_would_launch(pos0, nt, hd, nh, nkv, mailbox.numel()))


def attn_f16_mailbox(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int, nh: int, nkv: int,
                     mailbox: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
                     scratch: torch.Tensor | None = None) -> torch.Tensor:
    """attn_f16 with decode in one launch through `mailbox` (attn_mailbox) where the
    geometry allows it; otherwise the same as attn_f16 with `scratch`."""
    _need(q, torch.float32, "q")
    nt = q.shape[0]
    hd = q.shape[-1] // (2 * nh)
    kvd = nkv * hd
    if scale is None:
        scale = 1.0 / hd ** 0.5
    for c in (kc, vc):
        if c.dtype not in (torch.float16, torch.int16) or not c.is_contiguous() or c.shape[-1] != kvd:
            raise ValueError("kc/vc must be contiguous [ctx, nkv*hd] f16")
        if c.shape[0] < pos0 + nt:
            raise ValueError("cache shorter than pos0 + nt")
    if out is None:
        out = torch.empty(nt, nh * hd, device=q.device, dtype=torch.float32)
    _need(out, torch.float32, "out")
    if scratch is None:
        need = attn_scratch_bytes(pos0, nt, nh, nkv, hd)
        scratch = torch.empty(max(need, 1), device=q.device, dtype=torch.uint8)
    call("it_attn_f16_mailbox", q.data_ptr(), nh * 2 * hd, kc.data_ptr(), vc.data_ptr(), kvd, pos0, hd, nh, nkv, nt,
         float(scale), out.data_ptr(), nh * hd, mailbox.data_ptr(), mailbox.numel(), scratch.data_ptr(),
         scratch.numel(), _stream())
    return out


def _ckpt(ckpt, like: torch.Tensor):
    if ckpt is not None:
        _need(ckpt, torch.float32, "ckpt")
        if ckpt.numel() != like.numel():
            raise ValueError("ckpt must have the shape of the state it snapshots")


def gdn_conv(x: torch.Tensor, w: torch.Tensor, state: torch.Tensor, out: torch.Tensor | None = None,
             ckpt: torch.Tensor | None = None, ckpt_after: int = 0) -> torch.Tensor:
    """x [nt, cd] f32, w [cd, K], state [K-1, cd] (updated in place) -> silu(conv) [nt, cd].
    ckpt (optional, shape of state) receives the state after token ckpt_after."""
    _need(x, torch.float32, "x"); _need(w, torch.float32, "w"); _need(state, torch.float32, "state")
    _ckpt(ckpt, state)
    nt, cd = x.shape
    K = w.shape[1]
    if out is None:
        out = torch.empty_like(x)
    if ckpt is None:
        call("it_gdn_conv", x.data_ptr(), cd, w.data_ptr(), state.data_ptr(), out.data_ptr(), cd, cd, nt, K, _stream())
    else:
        call("it_gdn_conv_ckpt", x.data_ptr(), cd, w.data_ptr(), state.data_ptr(), out.data_ptr(), cd, cd, nt, K,
             ckpt.data_ptr(), ckpt_after, _stream())
    return out


def gdn_conv_l2norm(x: torch.Tensor, w: torch.Tensor, state: torch.Tensor, nnorm: int, eps: float = 1e-6,
                    out: torch.Tensor | None = None, ckpt: torch.Tensor | None = None,
                    ckpt_after: int = 0) -> torch.Tensor:
    """gdn_conv then l2norm_heads(out, nnorm, 128, eps) in one pass (x [nt, cd], cd % 128 == 0);
    ckpt as for gdn_conv."""
    _need(x, torch.float32, "x"); _need(w, torch.float32, "w"); _need(state, torch.float32, "state")
    _ckpt(ckpt, state)
    nt, cd = x.shape
    K = w.shape[1]
    if out is None:
        out = torch.empty_like(x)
    if ckpt is None:
        call("it_gdn_conv_l2norm", x.data_ptr(), cd, w.data_ptr(), state.data_ptr(), out.data_ptr(), cd, cd, nt, K,
             nnorm, float(eps), _stream())
    else:
        call("it_gdn_conv_l2norm_ckpt", x.data_ptr(), cd, w.data_ptr(), state.data_ptr(), out.data_ptr(), cd, cd, nt,
             K, nnorm, float(eps), ckpt.data_ptr(), ckpt_after, _stream())
    return out


def l2norm_heads(x: torch.Tensor, nheads: int, d: int, eps: float = 1e-6) -> torch.Tensor:
    """In place on the first nheads*d columns of each row of x [nt, C]."""
    _need(x, torch.float32, "x")
    call("it_l2norm_heads", x.data_ptr(), x.shape[1], nheads, d, x.shape[0], float(eps), _stream())
    return x


def gdn_decode_fused(x, w, conv_state_in, conv_state_out, beta_raw, alpha_raw, dt, a, state, nv: int, nk: int,
                     eps: float = 1e-6, out=None, ckpt_state=None, ckpt_conv=None, ckpt_after: int = 0):
    """One launch for a GDN decode layer (1 <= nt <= 4 tokens): gdn_conv_l2norm(x, w, ...) then
    gdn_step, with the conv state read from conv_state_in and the new one written to
    conv_state_out (a different buffer). x [nt, (2nk+nv)*128], state updated in place -> out
    [nt, nv*128]. ckpt_state / ckpt_conv (optional, together): both states after token ckpt_after
    (the MTP verify checkpoint)."""
    for t, n in ((x, "x"), (w, "w"), (conv_state_in, "conv_state_in"), (conv_state_out, "conv_state_out"),
                 (beta_raw, "beta_raw"), (alpha_raw, "alpha_raw"), (dt, "dt"), (a, "a"), (state, "state")):
        _need(t, torch.float32, n)
    nt, cd = x.shape
    S = state.shape[-1]
    if out is None:
        out = torch.empty(nt, nv * S, device=x.device, dtype=torch.float32)
    args = [x.data_ptr(), cd, w.data_ptr(), w.shape[1], conv_state_in.data_ptr(), conv_state_out.data_ptr(),
            beta_raw.data_ptr(), alpha_raw.data_ptr(), beta_raw.shape[1], dt.data_ptr(), a.data_ptr(), state.data_ptr(),
            out.data_ptr(), out.shape[1], nt, nv, nk, S, float(eps)]
    if ckpt_state is None and ckpt_conv is None:
        call("it_gdn_decode_fused", *args, _stream())
    else:
        _ckpt(ckpt_state, state)
        _ckpt(ckpt_conv, conv_state_in)
        call("it_gdn_decode_fused_ckpt", *args, ckpt_state.data_ptr(), ckpt_conv.data_ptr(), ckpt_after, _stream())
    return out


def gdn_step(co, beta_raw, alpha_raw, dt, a, state, nv: int, nk: int, out=None, chunked: bool = False,
             scratch=None, ckpt=None, ckpt_after: int = 0):
    """co [nt, (2nk+nv)S], beta_raw/alpha_raw [nt, nv], dt/a [nv], state [nv, S, S] (in place)
    -> out [nt, nv*S]. chunked=True uses the chunk-64 scan (it_gdn_chunked). ckpt (optional, shape
    of state; token-sequential kernel only) receives the state after token ckpt_after."""
    _ckpt(ckpt, state)
    if ckpt is not None and chunked:
        raise ValueError("the checkpoint is a feature of the token-sequential kernel")
    for t, n in ((co, "co"), (beta_raw, "beta_raw"), (alpha_raw, "alpha_raw"), (dt, "dt"), (a, "a"), (state, "state")):
        _need(t, torch.float32, n)
    nt = co.shape[0]
    S = state.shape[-1]
    if out is None:
        out = torch.empty(nt, nv * S, device=co.device, dtype=torch.float32)
    args = [co.data_ptr(), co.shape[1], beta_raw.data_ptr(), alpha_raw.data_ptr(), beta_raw.shape[1], dt.data_ptr(),
            a.data_ptr(), state.data_ptr(), out.data_ptr(), out.shape[1], nt, nv, nk, S]
    if chunked:
        need = lib().it_gdn_chunked_scratch_bytes(nt, nv, S)
        if scratch is None and need:
            scratch = torch.empty(need, device=co.device, dtype=torch.uint8)
        nbytes = 0 if scratch is None else scratch.numel() * scratch.element_size()
        call("it_gdn_chunked", *args, _ptr(scratch), nbytes, _stream())
    elif ckpt is not None:
        call("it_gdn_step_ckpt", *args, ckpt.data_ptr(), ckpt_after, _stream())
    else:
        call("it_gdn_step", *args, _stream())
    return out


def gdn_prefill(x, w, conv_state, beta_raw, alpha_raw, dt, a, state, nv: int, nk: int, eps: float = 1e-6, out=None,
                scratch=None):
    """The GDN layer over a prompt chunk in one call (it_gdn_prefill): conv + SiLU + q/k L2 kept as
    f16 in scratch, then the chunk-64 scan. x [nt, cd] f32, w [cd, K], conv_state [K-1, cd] and
    state [nv, S, S] updated in place -> out [nt, nv*S]."""
    for t, n in ((x, "x"), (w, "w"), (conv_state, "conv_state"), (beta_raw, "beta_raw"), (alpha_raw, "alpha_raw"),
                 (dt, "dt"), (a, "a"), (state, "state")):
        _need(t, torch.float32, n)
    nt = x.shape[0]
    S = state.shape[-1]
    if out is None:
        out = torch.empty(nt, nv * S, device=x.device, dtype=torch.float32)
    need = lib().it_gdn_prefill_scratch_bytes(nt, nv, nk, S)
    if scratch is None and need:
        scratch = torch.empty(need, device=x.device, dtype=torch.uint8)
    nbytes = 0 if scratch is None else scratch.numel() * scratch.element_size()
    call("it_gdn_prefill", x.data_ptr(), x.shape[1], w.data_ptr(), w.shape[1], conv_state.data_ptr(),
         beta_raw.data_ptr(), alpha_raw.data_ptr(), beta_raw.shape[1], dt.data_ptr(), a.data_ptr(), state.data_ptr(),
         out.data_ptr(), out.shape[1], nt, nv, nk, S, float(eps), _ptr(scratch), nbytes, _stream())
    return out


def gdn_gated_rmsnorm(o: torch.Tensor, z: torch.Tensor, w: torch.Tensor, nv: int, eps: float = 1e-6,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """o, z [nt, nv*128], w [128] -> o / rms(o) * w * silu(z) per 128-wide head row (out may be o)."""
    _need(o, torch.float32, "o"); _need(z, torch.float32, "z"); _need(w, torch.float32, "w")
    if out is None:
        out = torch.empty_like(o)
    call("it_gdn_gated_rmsnorm", o.data_ptr(), o.shape[1], z.data_ptr(), z.shape[1], w.data_ptr(), float(eps),
         out.data_ptr(), out.shape[1], nv, 128, o.shape[0], _stream())
    return out


def gdn_step_gated(co, beta_raw, alpha_raw, dt, a, state, nv: int, nk: int, z=None, norm_w=None, eps: float = 1e-6,
                   out=None, ckpt=None, ckpt_after: int = 0):
    """The recurrence with one workgroup per V head and, when z is given, the gated RMSNorm
    (o / rms(o) * norm_w * silu(z)) fused into the output write (it_gdn_step_gated)."""
    for t, n in ((co, "co"), (beta_raw, "beta_raw"), (alpha_raw, "alpha_raw"), (dt, "dt"), (a, "a"), (state, "state")):
        _need(t, torch.float32, n)
    if z is not None:
        _need(z, torch.float32, "z"); _need(norm_w, torch.float32, "norm_w")
    _ckpt(ckpt, state)
    nt = co.shape[0]
    S = state.shape[-1]
    if out is None:
        out = torch.empty(nt, nv * S, device=co.device, dtype=torch.float32)
    call("it_gdn_step_gated", co.data_ptr(), co.shape[1], beta_raw.data_ptr(), alpha_raw.data_ptr(), beta_raw.shape[1],
         dt.data_ptr(), a.data_ptr(), state.data_ptr(), out.data_ptr(), out.shape[1], nt, nv, nk, S, _ptr(z),
         0 if z is None else z.shape[1], _ptr(norm_w), float(eps), _ptr(ckpt), ckpt_after, _stream())
    return out


def gdn_rollback(ck_conv: torch.Tensor | None, conv_state: torch.Tensor | None, ck_ssm: torch.Tensor | None,
                 ssm: torch.Tensor | None) -> None:
    """Restore the checkpointed conv and SSM states after a rejected draft (it_gdn_rollback)."""
    cw = 0 if conv_state is None else conv_state.numel()
    sw = 0 if ssm is None else ssm.numel()
    for c, t in ((ck_conv, conv_state), (ck_ssm, ssm)):
        if t is not None and (c is None or c.numel() != t.numel()):
            raise ValueError("checkpoint and state sizes differ")
    call("it_gdn_rollback", _ptr(ck_conv), _ptr(conv_state), cw, _ptr(ck_ssm), _ptr(ssm), sw, _stream())


# ---- verification of a drafted token tree (include/it_attn.h has the whole contract)

ROPE_KINDS = {"plain": 0, "linear": 1, "ntk": 2, "yarn": 3}
ROPE_LAYOUTS = {"half": 0, "interleaved": 1}
TREE_MAX = 64


def _call_on(dev: int, name: str, *args) -> None:
    """call(name, *args, stream) with device dev current and its current stream (asked for as numbers: the stream
    object of torch.cuda.current_stream takes 1 us to make, a third of a short launch)."""
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            call(name, *args, torch._C._cuda_getCurrentRawStream(dev))
    elif getattr(lib(), name)(*args, torch._C._cuda_getCurrentRawStream(dev)):
        raise ItError(f"{name}: {last_error()}")


def _need_all(dtype: torch.dtype, dev: int, tensors, names: str) -> None:
    """Every tensor (None: absent) contiguous, of dtype and on device dev; names in the tensors' order, for the message.
    One pass over cheap queries: these checks are most of what a short call costs the host."""
    for t in tensors:
        if t is not None and (t.dtype is not dtype or t.get_device() != dev or dev < 0 or not t.is_contiguous()):
            name = names.split()[[u is t for u in tensors].index(True)]
            _need(t, dtype, name)
            raise ValueError(f"{name} must be on the same device as the other tensors")


def _need_caches(dtypes, dev: int, kvd: int, rows: int, kc: torch.Tensor, vc: torch.Tensor) -> None:
    for c in (kc, vc):
        shape = c.shape
        if c.dtype not in dtypes or len(shape) != 2 or shape[1] != kvd or not c.is_contiguous():
            raise ValueError(f"kc and vc must be contiguous [rows, {kvd}] of {dtypes[0]}")
        if c.get_device() != dev or dev < 0:
            raise ValueError("kc and vc must be device tensors, on the same device as the other tensors")
        if shape[0] < rows:
            raise ValueError(f"cache too short: {shape[0]} rows, {rows} needed")


_F16 = (torch.float16, torch.int16)
_F32 = (torch.float32,)


def rope_freqs(n_rot: int, base: float = 1e7, kind: str = "plain", factor: float = 1.0, orig_ctx: int = 8192,
               device="cuda") -> tuple[torch.Tensor, float]:
    """(freq [n_rot/2] f32 on device, mscale) for attn_prep_pos_*: plain, linear, ntk or yarn scaling of the context
    by factor (it_rope_freqs)."""
    if kind not in ROPE_KINDS:
        raise ValueError(f"kind must be one of {sorted(ROPE_KINDS)}")
    freq, m = torch.empty(max(n_rot // 2, 1), dtype=torch.float32), ctypes.c_float()
    call("it_rope_freqs", n_rot, float(base), ROPE_KINDS[kind], float(factor), orig_ctx, freq.data_ptr(),
         ctypes.addressof(m))
    return freq.to(device), m.value


def _prep_pos(name, kinds, q, k, v, kc, vc, pos, row0, nh, nkv, freq, mscale, layout, q_norm, k_norm, eps, pos0, *more):
    dev = q.get_device()
    _need_all(torch.float32, dev, (q, k, v, freq, q_norm, k_norm), "q k v freq q_norm k_norm")
    shape = k.shape
    if len(shape) != 2 or shape[1] % nkv != 0:
        raise ValueError("k must be [nt, nkv*hd]")
    nt, kvd = shape
    hd = kvd // nkv
    if q.shape != (nt, nh * 2 * hd) or v.shape != shape:
        raise ValueError("q must be [nt, nh*2*hd] and v the shape of k [nt, nkv*hd]")
    if row0 < 0:
        raise ValueError("row0 must not be negative")
    _need_caches(kinds, dev, kvd, row0 + nt, kc, vc)
    if pos is not None and (pos.shape != (nt,) or pos.dtype is not torch.int32 or pos.get_device() != dev or
                            not pos.is_contiguous()):
        _need_all(torch.int32, dev, (pos,), "pos")
        raise ValueError("pos must be [nt]")
    if (q_norm is not None and q_norm.numel() != hd) or (k_norm is not None and k_norm.numel() != hd):
        raise ValueError("q_norm and k_norm must hold head_dim floats")
    if layout not in ROPE_LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(ROPE_LAYOUTS)}")
    _call_on(dev, name, q.data_ptr(), nh * 2 * hd, k.data_ptr(), v.data_ptr(), kvd, _ptr(q_norm), _ptr(k_norm), eps,
             kc.data_ptr(), vc.data_ptr(), kvd, _ptr(pos), pos0, row0, hd, nh, nkv, nt, 2 * freq.numel(),
             freq.data_ptr(), mscale, ROPE_LAYOUTS[layout], *more)


def attn_prep_pos_f16(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor,
                      pos: torch.Tensor | None, row0: int, nh: int, nkv: int, freq: torch.Tensor, mscale: float = 1.0,
                      layout: str = "half", q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                      eps: float = 1e-6, round_mode: int = 0, pos0: int = 0) -> None:
    """attn_prep_f16 at given positions: token t at pos[t] int32 (None: pos0 + t), its K/V to cache row row0 + t, the
    first 2 * freq.numel() dims of each head turned by pos * freq[i] in pairs (i, i + n/2) ("half") or (2i, 2i + 1)
    ("interleaved"), cos and sin times mscale (it_attn_prep_pos_f16; freq and mscale from rope_freqs)."""
    _prep_pos("it_attn_prep_pos_f16", _F16, q, k, v, kc, vc, pos, row0, nh, nkv, freq, mscale, layout, q_norm, k_norm, eps,
              pos0, round_mode)


def attn_prep_pos_f32kv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor,
                        pos: torch.Tensor | None, row0: int, nh: int, nkv: int, freq: torch.Tensor, mscale: float = 1.0,
                        layout: str = "half", q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                        eps: float = 1e-6, pos0: int = 0) -> None:
    """attn_prep_pos_f16 for the MTP head's f32 cache (it_attn_prep_pos_f32kv)."""
    _prep_pos("it_attn_prep_pos_f32kv", _F32, q, k, v, kc, vc, pos, row0, nh, nkv, freq, mscale, layout, q_norm, k_norm, eps,
              pos0)


def _need_anc(anc: torch.Tensor, dev: int, nt: int) -> None:
    if anc.shape != (nt,) or anc.dtype is not torch.int64 or anc.get_device() != dev or not anc.is_contiguous():
        _need_all(torch.int64, dev, (anc,), "anc")
        raise ValueError(f"anc must be [{nt}]")


def tree_plan(parent: torch.Tensor, p0: int) -> tuple[torch.Tensor, torch.Tensor]:
    """parent [nt] int32 (-1: follows the last committed token; outside -1 .. t-1: padding) -> (anc [nt] int64, the
    bits of each node and its ancestors, pos [nt] int32 = p0 + depth) (it_tree_plan)."""
    _need(parent, torch.int32, "parent")
    nt = parent.numel()
    anc = torch.empty(nt, device=parent.device, dtype=torch.int64)
    pos = torch.empty(nt, device=parent.device, dtype=torch.int32)
    _call_on(parent.get_device(), "it_tree_plan", parent.data_ptr(), nt, p0, anc.data_ptr(), pos.data_ptr())
    return anc, pos


def attn_tree_scratch_bytes(pos0: int, nt: int, nh: int, nkv: int, hd: int = 256) -> int:
    return lib().it_attn_tree_scratch_bytes(pos0, nt, hd, nh, nkv)


def attn_tree_f32kv_scratch_bytes(pos0: int, nt: int, nh: int, nkv: int, hd: int = 256) -> int:
    return lib().it_attn_tree_f32kv_scratch_bytes(pos0, nt, hd, nh, nkv)


def _attn_tree(name, kinds, scratch_bytes, q, kc, vc, pos0, nh, nkv, anc, scale, out, scratch, rows):
    dev, shape = q.get_device(), q.shape
    if len(shape) != 2 or shape[1] % (2 * nh) != 0:
        raise ValueError("q must be [nt, nh*2*hd]")
    nt, hd = shape[0], shape[1] // (2 * nh)
    kvd = nkv * hd
    if rows is None:
        rows = nt
    if out is None:
        out = torch.empty(nt, nh * hd, device=q.device, dtype=torch.float32)
    _need_all(torch.float32, dev, (q, out), "q out")
    if out.shape != (nt, nh * hd):
        raise ValueError("out must be [nt, nh*hd]")
    _need_caches(kinds, dev, kvd, pos0 + rows, kc, vc)
    _need_anc(anc, dev, nt)
    if scale is None:
        scale = 1.0 / hd ** 0.5
    if scratch is None:
        need = scratch_bytes(pos0, nt, nh, nkv, hd)
        scratch = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
    elif scratch.get_device() != dev or not scratch.is_contiguous():
        raise ValueError("scratch must be contiguous, on the same device as the other tensors")
    nbytes = 0 if scratch is None else scratch.nbytes
    _call_on(dev, name, q.data_ptr(), nh * 2 * hd, kc.data_ptr(), vc.data_ptr(), kvd, pos0, hd, nh, nkv, nt, rows,
             anc.data_ptr(), scale, out.data_ptr(), nh * hd, _ptr(scratch), nbytes)
    return out


def attn_tree_f16(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int, nh: int, nkv: int, anc: torch.Tensor,
                  scale: float | None = None, out: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
                  rows: int | None = None) -> torch.Tensor:
    """attn_f16 for nodes of a drafted tree: q [nt, nh*2*hd] f32, the tree's `rows` nodes (None: nt, all of them) in cache
    rows pos0 + j, anc [nt] int64 (tree_plan) the nodes that each query sees -> out [nt, nh*hd] f32; zeros for padding
    nodes (it_attn_tree_f16)."""
    return _attn_tree("it_attn_tree_f16", _F16, attn_tree_scratch_bytes, q, kc, vc, pos0, nh, nkv, anc, scale, out, scratch,
                      rows)


def attn_tree_f32kv(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos0: int, nh: int, nkv: int, anc: torch.Tensor,
                    scale: float | None = None, out: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
                    rows: int | None = None) -> torch.Tensor:
    """attn_tree_f16 over the MTP head's f32 cache (it_attn_tree_f32kv)."""
    return _attn_tree("it_attn_tree_f32kv", _F32, attn_tree_f32kv_scratch_bytes, q, kc, vc, pos0, nh, nkv, anc, scale, out,
                      scratch, rows)


def _kv_tree_commit(name, kinds, kc, vc, pos0, nt, anc, leaf):
    dev = kc.get_device()
    if dev < 0 or kc.dim() != 2:
        raise ValueError("kc must be a device tensor [rows, kvd]")
    if vc.dtype is not kc.dtype:
        raise ValueError("kc and vc must have one dtype")
    kvd = kc.shape[1]
    _need_caches(kinds, dev, kvd, pos0 + nt, kc, vc)
    _need_anc(anc, dev, nt)
    _call_on(dev, name, kc.data_ptr(), vc.data_ptr(), kvd, pos0, nt, anc.data_ptr(), leaf)


def kv_tree_commit_f16(kc: torch.Tensor, vc: torch.Tensor, pos0: int, nt: int, anc: torch.Tensor, leaf: int) -> None:
    """Moves the cache rows of node leaf's path (rows pos0 + t hold the nodes) to rows pos0, pos0 + 1, ...; leaf -1:
    nothing (it_kv_tree_commit_f16)."""
    _kv_tree_commit("it_kv_tree_commit_f16", _F16, kc, vc, pos0, nt, anc, leaf)


def kv_tree_commit_f32(kc: torch.Tensor, vc: torch.Tensor, pos0: int, nt: int, anc: torch.Tensor, leaf: int) -> None:
    """kv_tree_commit_f16 for the MTP head's f32 cache."""
    _kv_tree_commit("it_kv_tree_commit_f32", _F32, kc, vc, pos0, nt, anc, leaf)


def gdn_tree_trace(nt: int, nv: int, nk: int, device) -> torch.Tensor:
    """A buffer for what gdn_tree leaves to gdn_tree_commit: one per layer, for trees of up to nt nodes."""
    return torch.empty(lib().it_gdn_tree_trace_bytes(nt, nv, nk, 128), device=device, dtype=torch.uint8)


def gdn_tree(x: torch.Tensor, w: torch.Tensor, conv_state: torch.Tensor, beta_raw: torch.Tensor, alpha_raw: torch.Tensor,
             dt: torch.Tensor, a: torch.Tensor, state: torch.Tensor, anc: torch.Tensor, nv: int, nk: int,
             trace: torch.Tensor, eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """The recurrent layer over a drafted tree in one launch: x [nt, (2nk+nv)*128], w [cd, K], conv_state [K-1, cd] and
    state [nv, 128, 128] (both only read), beta_raw/alpha_raw [nt, nv], anc [nt] int64 (tree_plan) -> out
    [nt, nv*128]; trace (gdn_tree_trace) keeps what gdn_tree_commit needs (it_gdn_tree)."""
    dev, (nt, cd), K = x.get_device(), x.shape, conv_state.shape[0] + 1
    if out is None:
        out = torch.empty(nt, nv * 128, device=x.device, dtype=torch.float32)
    _need_all(torch.float32, dev, (x, conv_state, state, w, beta_raw, alpha_raw, dt, a, out),
              "x conv_state state w beta_raw alpha_raw dt a out")
    if cd != (2 * nk + nv) * 128 or conv_state.shape != (K - 1, cd) or state.shape != (nv, 128, 128):
        raise ValueError("x must be [nt, (2nk+nv)*128], conv_state [K-1, (2nk+nv)*128] and state [nv, 128, 128]")
    if w.shape != (cd, K) or beta_raw.shape != (nt, nv) or alpha_raw.shape != (nt, nv) or dt.numel() != nv or \
            a.numel() != nv or out.shape != (nt, nv * 128):
        raise ValueError("w must be [cd, K], beta_raw / alpha_raw [nt, nv], dt / a [nv] and out [nt, nv*128]")
    _need_anc(anc, dev, nt)
    _need_all(torch.uint8, dev, (trace,), "trace")
    _call_on(dev, "it_gdn_tree", x.data_ptr(), cd, w.data_ptr(), K, conv_state.data_ptr(), beta_raw.data_ptr(),
             alpha_raw.data_ptr(), nv, dt.data_ptr(), a.data_ptr(), state.data_ptr(), anc.data_ptr(), out.data_ptr(),
             nv * 128, nt, nv, nk, 128, eps, trace.data_ptr(), trace.numel())
    return out


def gdn_tree_commit(x: torch.Tensor, conv_state: torch.Tensor, state: torch.Tensor, anc: torch.Tensor, leaf: int, nv: int,
                    nk: int, trace: torch.Tensor) -> None:
    """conv_state and state <- those after node leaf of the gdn_tree call that wrote trace (the same x and anc); leaf -1:
    they stay (it_gdn_tree_commit)."""
    dev, (nt, cd), K = x.get_device(), x.shape, conv_state.shape[0] + 1
    _need_all(torch.float32, dev, (x, conv_state, state), "x conv_state state")
    if cd != (2 * nk + nv) * 128 or conv_state.shape != (K - 1, cd) or state.shape != (nv, 128, 128):
        raise ValueError("x must be [nt, (2nk+nv)*128], conv_state [K-1, (2nk+nv)*128] and state [nv, 128, 128]")
    _need_anc(anc, dev, nt)
    _need_all(torch.uint8, dev, (trace,), "trace")
    _call_on(dev, "it_gdn_tree_commit", x.data_ptr(), cd, K, conv_state.data_ptr(), state.data_ptr(), anc.data_ptr(), leaf,
             nt, nv, nk, 128, trace.data_ptr(), trace.numel())


# ---- a paged K/V cache in 8 bits (include/it_attn.h has the whole contract)

KV8_PAGE, KV8_BLOCK = 64, 16


class Kv8Cache(NamedTuple):
    """A layer's buffers: codes kp, vp [npages, nkv, 64*hd] uint8, scales sc [npages, nkv, 8] f16, open rows tk, tv
    [nseq, 2, nkv, 64*hd] f16 (it_kv8_cache)."""
    kp: torch.Tensor
    vp: torch.Tensor
    sc: torch.Tensor
    tk: torch.Tensor
    tv: torch.Tensor


def kv8_cache(npages: int, nseq: int, nkv: int, hd: int = 256, device="cuda") -> Kv8Cache:
    """A cache of npages pages of 64 rows, for nseq sequences. What it holds before the first append does not matter."""
    def new(dtype, *shape):
        return torch.zeros(*shape, dtype=dtype, device=device)
    return Kv8Cache(new(torch.uint8, npages, nkv, KV8_PAGE * hd), new(torch.uint8, npages, nkv, KV8_PAGE * hd),
                    new(torch.float16, npages, nkv, 8), new(torch.float16, nseq, 2, nkv, KV8_PAGE * hd),
                    new(torch.float16, nseq, 2, nkv, KV8_PAGE * hd))


def _kv8(c: Kv8Cache):
    """(device, nkv, hd, nseq, it_kv8_cache) of a cache whose buffers fit each other. (The checks of these calls are most of
    what a short one costs the host: one expression over cheap queries, and messages only once it fails.)"""
    kp, vp, sc, tk, tv = c
    dev, shape, tail = kp.get_device(), kp.shape, tk.shape
    if len(shape) != 3 or len(tail) != 4 or shape[2] % KV8_PAGE:
        raise ValueError("kp must be [npages, nkv, 64*hd] and tk [nseq, 2, nkv, 64*hd]")
    npages, nkv, size = shape
    if vp.shape != shape or sc.shape != (npages, nkv, 8) or tail[1:] != (2, nkv, size) or tv.shape != tail:
        raise ValueError("vp must have kp's shape, sc [npages, nkv, 8], tk and tv [nseq, 2, nkv, 64*hd]")
    if not (dev >= 0 and kp.dtype is torch.uint8 and vp.dtype is torch.uint8 and sc.dtype is torch.float16 and
            tk.dtype is torch.float16 and tv.dtype is torch.float16 and vp.get_device() == dev and sc.get_device() == dev and
            tk.get_device() == dev and tv.get_device() == dev and kp.is_contiguous() and vp.is_contiguous() and
            sc.is_contiguous() and tk.is_contiguous() and tv.is_contiguous()):
        _need_all(torch.uint8, dev, (kp, vp), "kp vp")
        _need_all(torch.float16, dev, (sc, tk, tv), "sc tk tv")
    hd = size // KV8_PAGE
    return dev, nkv, hd, tail[0], Kv8CacheArgs(kp.data_ptr(), vp.data_ptr(), sc.data_ptr(), tk.data_ptr(), tv.data_ptr(),
                                               npages, tail[0], nkv, hd)


def _kv8_batch(dev: int, nseq: int, start: torch.Tensor, length: torch.Tensor, table: torch.Tensor) -> int:
    shape = table.shape
    if not (start.dtype is torch.int32 and length.dtype is torch.int32 and table.dtype is torch.int32 and
            start.get_device() == dev and length.get_device() == dev and table.get_device() == dev and
            start.is_contiguous() and length.is_contiguous() and table.is_contiguous()):
        _need_all(torch.int32, dev, (start, length, table), "start length table")
    if start.shape != (nseq + 1,) or length.shape != (nseq,) or len(shape) != 2 or shape[0] != nseq:
        raise ValueError(f"start must be [{nseq + 1}], length [{nseq}] and table [{nseq}, max_pages]: one of each for the "
                         "cache's sequences")
    return shape[1]


def _kv8_rows(dev: int, kvd: int, k: torch.Tensor, v: torch.Tensor) -> int:
    """Token stride of f16 rows k, v [ntok, kvd]; rows may lie apart, as a slice of wider ones."""
    shape, step = k.shape, k.stride()
    if not (k.dtype is torch.float16 and v.dtype is torch.float16 and k.get_device() == dev and v.get_device() == dev and
            len(shape) == 2 and shape[1] == kvd):
        raise ValueError(f"k and v must be [ntok, {kvd}] f16 on the cache's device")
    if v.shape != shape or v.stride() != step or step[1] != 1:
        raise ValueError("k and v must have one shape and one stride, with each row's values side by side")
    return step[0]


def kv8_append(cache: Kv8Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, length: torch.Tensor,
               table: torch.Tensor, max_nt: int) -> None:
    """Appends f16 rows k, v [ntok, nkv*hd]: rows start[i] .. start[i+1]-1 follow the length[i] rows that sequence i holds
    (start [nseq+1], length [nseq], table [nseq, max_pages] int32 on the device; at most max_nt a sequence). Pages that
    get full are quantised; length stays as it is (it_kv8_append). Up to 64 of a call's own rows are taken back by a smaller length;
    further back by the rule of it_attn.h alone, or by kv8_read and appending anew."""
    dev, nkv, hd, nseq, args = _kv8(cache)
    pages = _kv8_batch(dev, nseq, start, length, table)
    stride = _kv8_rows(dev, nkv * hd, k, v)
    _call_on(dev, "it_kv8_append", ctypes.addressof(args), k.data_ptr(), v.data_ptr(), stride, k.shape[0],
             start.data_ptr(), length.data_ptr(), table.data_ptr(), pages, max_nt)


def kv8_read(cache: Kv8Cache, start: torch.Tensor, first: torch.Tensor, total: torch.Tensor, table: torch.Tensor,
             max_rows: int, rows: int, out: tuple[torch.Tensor, torch.Tensor] | None = None
             ) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows first[i] .. of the sequences as f16 k, v [rows, nkv*hd], start[i+1] - start[i] (at most max_rows) of sequence
    i at row start[i]; total [nseq] the rows that each one holds (it_kv8_read). Rows that no sequence has are left as they are
    in out, the tensors to write to; rows that cannot be (a negative first or total, more than the table can name) are NaN."""
    dev, nkv, hd, nseq, args = _kv8(cache)
    pages = _kv8_batch(dev, nseq, start, total, table)
    if first.shape != (nseq,):
        raise ValueError(f"first must be [{nseq}]")
    if first.dtype is not torch.int32 or first.get_device() != dev or not first.is_contiguous():
        _need_all(torch.int32, dev, (first,), "first")
    if out is None:
        at = cache.kp.device
        out = (torch.empty(rows, nkv * hd, dtype=torch.float16, device=at), torch.empty(rows, nkv * hd, dtype=torch.float16, device=at))
    k, v = out
    stride = _kv8_rows(dev, nkv * hd, k, v)
    if k.shape[0] != rows:
        raise ValueError(f"out must be two of [{rows}, {nkv * hd}]")
    _call_on(dev, "it_kv8_read", ctypes.addressof(args), k.data_ptr(), v.data_ptr(), stride, rows, start.data_ptr(),
             first.data_ptr(), total.data_ptr(), table.data_ptr(), pages, max_rows)
    return k, v


def kv8_copy(cache: Kv8Cache, src: torch.Tensor | None = None, dst: torch.Tensor | None = None,
             seq_src: torch.Tensor | None = None, seq_dst: torch.Tensor | None = None) -> None:
    """Copies pages src[i] to dst[i] and the open rows of sequences seq_src[i] to seq_dst[i] (int32 on the device; no
    destination twice, and none that is a source) (it_kv8_copy)."""
    dev, _, _, _, args = _kv8(cache)
    for a, b in ((src, dst), (seq_src, seq_dst)):
        if (a is None) != (b is None) or (a is not None and (len(a.shape) != 1 or a.shape != b.shape)):
            raise ValueError("src and dst, seq_src and seq_dst must be pairs of one length")
    _need_all(torch.int32, dev, (src, dst, seq_src, seq_dst), "src dst seq_src seq_dst")
    _call_on(dev, "it_kv8_copy", ctypes.addressof(args), _ptr(src), _ptr(dst), 0 if src is None else len(src), _ptr(seq_src),
             _ptr(seq_dst), 0 if seq_src is None else len(seq_src))


@functools.lru_cache(maxsize=256)
def attn_kv8_scratch_bytes(max_nt: int, nh: int, nkv: int, hd: int = 256) -> int:
    return lib().it_attn_kv8_scratch_bytes(max_nt, hd, nh, nkv)


def attn_kv8(cache: Kv8Cache, q: torch.Tensor, start: torch.Tensor, length: torch.Tensor, table: torch.Tensor, nh: int,
             max_nt: int, scale: float | None = None, out: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
             out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Attention of appended tokens over the cache: q [ntok, nh*2*hd] f32 (q | gate per head), token t of sequence i sees its
    rows 0 .. length[i] + t -> out [ntok, nh*hd], f32 or f16 (out's type, or out_dtype). start, length, table, max_nt as for
    kv8_append, length still without the new tokens: with them all rows that the sequence holds, or fewer that it may be cut to
    (it_attn_kv8). An f16 output of more than 16 query rows of a KV head (max_nt times its heads) is not the f32 one rounded:
    probabilities go into its products as one f16 and q with two digits in place of three, which costs up to 2.1e-4 of the result in
    the mean beside the rounding's 2.1e-4."""
    dev, nkv, hd, nseq, args = _kv8(cache)
    pages = _kv8_batch(dev, nseq, start, length, table)
    shape, width = q.shape, nh * hd
    ntok = shape[0]
    if len(shape) != 2 or shape[1] != 2 * width:
        raise ValueError(f"q must be [ntok, {2 * width}]")
    if q.dtype is not torch.float32 or q.get_device() != dev or not q.is_contiguous():
        _need_all(torch.float32, dev, (q,), "q")
    if out is None:
        out = torch.empty(ntok, width, dtype=out_dtype, device=q.device)
    kind = out.dtype
    if (kind is not torch.float32 and kind is not torch.float16) or out.shape != (ntok, width):
        raise ValueError(f"out must be [{ntok}, {width}] of float32 or float16")
    if out.get_device() != dev or not out.is_contiguous():
        _need_all(kind, dev, (out,), "out")
    if scale is None:
        scale = 1.0 / hd ** 0.5
    if scratch is None:
        scratch = torch.empty(attn_kv8_scratch_bytes(max_nt, nh, nkv, hd), dtype=torch.uint8, device=q.device)
    elif scratch.get_device() != dev or not scratch.is_contiguous():
        raise ValueError("scratch must be contiguous, on the same device as the other tensors")
    _call_on(dev, "it_attn_kv8", ctypes.addressof(args), q.data_ptr(), 2 * width, ntok, start.data_ptr(), length.data_ptr(),
             table.data_ptr(), pages, max_nt, nh, scale, out.data_ptr(), width, kind is torch.float16, scratch.data_ptr(),
             scratch.nbytes)
    return out

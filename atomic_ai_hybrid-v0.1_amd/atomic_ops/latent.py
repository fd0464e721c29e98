"""PyTorch host side of latent attention: attention whose keys and values come
from one latent vector a token.  Every computation runs in libatomic_hybrid.so;
there is no fallback.

Sizes: H heads; dn, the key width without position; dr, the rotated key width
(shared by all heads); dv, the value width; dc, the latent width.  ``w_kv``
[H, dn + dv, dc] is the up-projection, as a Linear layer from dc to H (dn + dv)
holds it.  Operands are bfloat16 or float32 (one dtype).

Expanded form (prompts and training): ``kv`` [B, S, H, dn + dv] is the
up-projection's output and ``k_pe`` [B, S, dr] the rotated key.
  ``attention``           differentiable in q, kv and k_pe
  ``forward``/``backward``  the two directions by themselves, outside any graph
Absorbed form (single tokens, or a few a sequence), over the latents of a paged
cache [pages, page, dc + dr] whose rows are [latent | rotated key]:
  ``append``   writes tokens into the cache and rotates keys and queries
  ``decode``   reads it
The two forms of the same weights and tokens give the same outputs up to rounding.
No queries, keys or tokens (a dimension of zero) give empty or zero outputs.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DT = {torch.float32: _lib.ATOMIC_F32, torch.bfloat16: _lib.ATOMIC_BF16}


_MOST_ROW_BYTES = 1 << 25
_PIECE = {torch.float32: 3, torch.bfloat16: 7}   # elements of a 16-byte piece, less one


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _strided(t, n):
    """``(tensor, strides)``: t as the library reads it, with its first n
    strides (that of a dimension of one is never stepped along).  The last dimension has to be dense and
    the strides and the address whole 16-byte pieces; anything else is copied.
    Every other order of the first dimensions is read in place."""
    mask = _PIECE[t.dtype]
    for _ in range(2):
        s, odd = t.stride(), t.data_ptr() & 15
        if s[-1] == 1 and not odd and not any(x & mask for x in s[:n]):
            return t, s[:n]
        shape = t.shape
        s = tuple(s[i] if shape[i] > 1 else 0 for i in range(n))
        if (shape[-1] == 1 or t.stride(-1) == 1) and not odd and not any(x & mask for x in s):
            return t, s
        t = t.clone() if t.is_contiguous() else t.contiguous()
    raise ValueError("latent attention: rows have to be whole 16-byte pieces (dimensions that are multiples of 8)")


def _in_graph(*ts):
    """Whether a call with these tensors belongs to a graph."""
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _tangents(*ts):
    """Whether any of the tensors carries a forward-mode tangent.  (The level by
    itself first, as unpack_dual does: 1.5 us less of a call of 18.)"""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts)


def _operands(what, *named):
    """Checks that the operands are on one HIP device and of one supported dtype."""
    name0, first = named[0]
    if not first.is_cuda:
        raise ValueError(f"{what}: inputs must be HIP device tensors")
    dtype, device = first.dtype, first.get_device()
    if dtype not in _DT:
        raise TypeError(f"{what}: {name0} must be bfloat16 or float32")
    for name, t in named[1:]:
        if t.get_device() != device:
            raise ValueError(f"{what}: {name} must be on {name0}'s device")
        if t.dtype != dtype:
            raise TypeError(f"{what}: {name} must have {name0}'s dtype")


def _index(what, name, t, shape, dtype, device):
    if t.dtype != dtype or t.shape != shape or t.get_device() != device:
        raise ValueError(f"{what}: {name} must be {str(dtype)[6:]} {list(shape)} on the inputs' device")
    return t if t.is_contiguous() else t.contiguous()


def _workspace(ws, nbytes, device):
    """The caller's workspace where it is large enough, else a new one."""
    if ws is None or ws.numel() < nbytes:
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    if ws.device != device or ws.dtype != torch.uint8 or not ws.is_contiguous():
        raise ValueError("latent attention: workspace must be dense uint8 on the inputs' device")
    return ws


# ------------------------------------------------------------ expanded form
def _check(q, kv, k_pe, q_lens, kv_lens):
    _operands("latent attention", ("q", q), ("kv", kv), ("k_pe", k_pe))
    if q.dim() != 4 or kv.dim() != 4 or k_pe.dim() != 3:
        raise ValueError("q must be [B, T, H, dn + dr], kv [B, S, H, dn + dv] and k_pe [B, S, dr]")
    B, T, H, d = q.shape
    S, dr = k_pe.shape[1:]
    if kv.shape[:3] != (B, S, H) or k_pe.shape[0] != B or not 0 < dr < d or kv.shape[3] <= d - dr:
        raise ValueError("q must be [B, T, H, dn + dr], kv [B, S, H, dn + dv] and k_pe [B, S, dr]")
    if q_lens is not None:
        q_lens = _index("latent attention", "q_lens", q_lens, (B,), torch.int32, q.get_device())
    if kv_lens is not None:
        kv_lens = _index("latent attention", "kv_lens", kv_lens, (B,), torch.int32, q.get_device())
    return q_lens, kv_lens


def _rows(t, n):
    """``_strided`` for [B, rows, ...]; rows more than 32 MB apart are copied too."""
    t, s = _strided(t, n)
    if s[1] * t.element_size() <= _MOST_ROW_BYTES:
        return t, s
    if t.shape[1] == 1:
        return t, (s[0], 0, *s[2:])
    return _strided(t.contiguous(), n)


def make_args(q, kv, k_pe, scale, causal, dout=None):
    """``(args, operands)``: the args struct and the operands as the library reads them."""
    B, T, H, d = q.shape
    S, dr = k_pe.shape[1:]
    q, qs = _rows(q, 3)
    kv, ks = _rows(kv, 3)
    k_pe, ps = _rows(k_pe, 2)
    gs = (0, 0, 0)
    if dout is not None:
        dout, gs = _rows(dout, 3)
    args = _lib.LatentArgs(B, T, S, H, d - dr, dr, kv.shape[3] - (d - dr), _DT[q.dtype], 1 if causal else 0, scale,
                           qs, ks, ps, gs)
    return args, (q, kv, k_pe, dout)


def forward(q, kv, k_pe, scale, *, causal=True, q_lens=None, kv_lens=None, save=False, workspace=None, timer=None):
    """``(o, lse)``: o [B, T, H, dv] in q's dtype and lse [B, H, T] float32.
    With ``save`` ``(o, lse, rest)``: rest, for ``backward``, is what o's rounding
    to bfloat16 left out (None in float32).

    Query i of batch row b sees the keys j < kv_lens[b]; with ``causal`` those
    with j <= i + kv_lens[b] - q_lens[b] (queries stand at the end of the keys).
    ``q_lens`` / ``kv_lens`` are int32 [B] on the device (the whole T / S without
    them).  A query that sees no key, and one past its length, has o = 0 and
    lse = -inf.  What lies past the lengths does not matter; within them an
    infinity or NaN in a token's values may reach queries that do not see it (a
    weight of zero times it).  Inputs of any batch, token and head strides are
    read in place."""
    q_lens, kv_lens = _check(q, kv, k_pe, q_lens, kv_lens)
    lib = _lib.load()
    if not (q.numel() and kv.numel()):      # no queries, or none that sees a key
        o = q.new_zeros(*q.shape[:3], kv.shape[3] - (q.shape[3] - k_pe.shape[2]))
        lse = q.new_full((q.shape[0], q.shape[2], q.shape[1]), float("-inf"), dtype=torch.float32)
        return (o, lse, torch.zeros_like(o) if q.dtype == torch.bfloat16 else None) if save else (o, lse)
    args, (q, kv, k_pe, _) = make_args(q, kv, k_pe, scale, causal)
    if timer is not None:
        args.profile = timer.arm()
    B, T, H = q.shape[:3]
    nbytes = lib.atomic_latent_fwd_workspace_size(ctypes.byref(args))
    if nbytes == 0:
        raise _lib.AtomicError("atomic_latent_fwd: ATOMIC_ERR_SHAPE: unsupported or inconsistent dimensions",
                               _lib.ATOMIC_ERR_SHAPE)
    workspace = _workspace(workspace, nbytes, q.device)
    o = torch.empty(B, T, H, args.dv, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, H, T, dtype=torch.float32, device=q.device)
    rest = torch.empty_like(o) if save and q.dtype == torch.bfloat16 else None
    rc = lib.atomic_latent_fwd(ctypes.byref(args), _ptr(q), _ptr(kv), _ptr(k_pe), _ptr(q_lens), _ptr(kv_lens),
                               _ptr(o), _ptr(lse), _ptr(rest), _ptr(workspace), workspace.numel(), _stream(q.device))
    _lib.check(rc, "atomic_latent_fwd")
    return (o, lse, rest) if save else (o, lse)


def backward(q, kv, k_pe, o, lse, dout, scale, *, causal=True, q_lens=None, kv_lens=None, rest=None, workspace=None,
             timer=None):
    """``(dq, dkv, dk_pe)`` in the inputs' shapes and dtype from the forward's
    ``o``, ``lse`` and ``rest``; k_pe's gradient is summed over the heads.  A
    score's gradient is a difference of do . v and do . o: without ``rest``, o's
    rounding is most of what is left where a query sees few keys; one that sees a
    single key gives its score a gradient of exactly zero.  The same inputs give the
    same bits."""
    q_lens, kv_lens = _check(q, kv, k_pe, q_lens, kv_lens)
    B, T, H, d = q.shape
    dv = kv.shape[3] - (d - k_pe.shape[2])
    _operands("latent attention", ("q", q), ("o", o), ("dout", dout))
    if o.shape != (B, T, H, dv) or dout.shape != o.shape:
        raise ValueError("o and dout must be [B, T, H, dv]")
    if rest is not None:
        _operands("latent attention", ("q", q), ("rest", rest))
        if rest.shape != o.shape:
            raise ValueError("rest must be [B, T, H, dv]")
        rest = rest.contiguous()
    if lse.shape != (B, H, T) or lse.dtype != torch.float32 or lse.get_device() != q.get_device():
        raise ValueError("lse must be float32 [B, H, T] on q's device")
    lib = _lib.load()
    if not (q.numel() and kv.numel()):
        return tuple(torch.zeros_like(t, memory_format=torch.contiguous_format) for t in (q, kv, k_pe))
    args, (q, kv, k_pe, dout) = make_args(q, kv, k_pe, scale, causal, dout)
    if timer is not None:
        args.profile = timer.arm()
    nbytes = lib.atomic_latent_bwd_workspace_size(ctypes.byref(args))
    if nbytes == 0:
        raise _lib.AtomicError("atomic_latent_bwd_workspace_size: unsupported shape")
    workspace = _workspace(workspace, nbytes, q.device)
    o, lse = o.contiguous(), lse.contiguous()
    dq, dkv, dk = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, kv, k_pe))
    rc = lib.atomic_latent_bwd(ctypes.byref(args), _ptr(q), _ptr(kv), _ptr(k_pe), _ptr(q_lens), _ptr(kv_lens),
                               _ptr(o), _ptr(lse), _ptr(rest), _ptr(dout), _ptr(dq), _ptr(dkv), _ptr(dk),
                               _ptr(workspace), workspace.numel(), _stream(q.device))
    _lib.check(rc, "atomic_latent_bwd")
    return dq, dkv, dk


class LatentAttention(torch.autograd.Function):
    """``forward`` with ``backward`` as its gradient."""

    @staticmethod
    def forward(ctx, q, kv, k_pe, scale, causal, q_lens, kv_lens):
        o, lse, rest = forward(q, kv, k_pe, scale, causal=causal, q_lens=q_lens, kv_lens=kv_lens, save=True)
        ctx.save_for_backward(q, kv, k_pe, o, lse, rest, q_lens, kv_lens)
        ctx.scale, ctx.causal = scale, causal
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, kv, k_pe, o, lse, rest, q_lens, kv_lens = ctx.saved_tensors
        dq, dkv, dk = backward(q, kv, k_pe, o, lse, dout.to(q.dtype), ctx.scale, causal=ctx.causal, q_lens=q_lens,
                               kv_lens=kv_lens, rest=rest)
        return dq, dkv, dk, None, None, None, None


def attention(q, kv, k_pe, scale, *, causal=True, q_lens=None, kv_lens=None):
    """o [B, T, H, dv] of ``forward``, differentiable in q, kv and k_pe (reverse
    mode; forward-mode tangents are refused)."""
    if not (_in_graph(q, kv, k_pe) or _tangents(q, kv, k_pe)):
        return forward(q, kv, k_pe, scale, causal=causal, q_lens=q_lens, kv_lens=kv_lens)[0]
    return LatentAttention.apply(q, kv, k_pe, scale, causal, q_lens, kv_lens)


# ------------------------------------------------------------ paged cache
def _tables(what, cos, sin, dr, device):
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or cos.shape[1] != dr // 2 or \
            cos.shape[0] < 1 or sin.shape != cos.shape or cos.get_device() != device or sin.get_device() != device:
        raise ValueError(f"{what}: cos and sin must be float32 [positions, dr / 2] on the inputs' device")
    return cos if cos.is_contiguous() else cos.contiguous(), sin if sin.is_contiguous() else sin.contiguous()


def _cache(what, cache, width):
    if cache.dim() != 3 or cache.shape[2] != width or not cache.is_contiguous() or cache.data_ptr() % 16:
        raise ValueError(f"{what}: cache must be a dense [pages, page, dc + dr]")


def append(cache, c_kv, k_pe, slots, positions, cos, sin, *, q=None, interleaved=False, timer=None):
    """Appends N tokens to the cache and rotates by position on the way.

    Row ``slots[t]`` (page slots[t] // page, row slots[t] % page; int64 [N])
    becomes [c_kv[t] | rotate(k_pe[t])]; a negative slot, or one past the cache,
    leaves it as it is.  Slots have to differ: the row of one that occurs twice is a
    mixture of the tokens' (a row is written by many threads, the tokens' in no order).
    ``positions`` int32 [N] choose the rows of the float32 tables ``cos`` / ``sin``
    [positions, dr / 2]; the rotation turns the pairs (i, i + dr / 2), or
    (2 i, 2 i + 1) with ``interleaved``.  Returns
    ``(k, q)``: the rotated keys [N, dr] and, where ``q`` [N, H, dn + dr] is
    given, q with its last dr elements rotated (else None).  ``cache`` None
    (with c_kv and slots None) only rotates.

    The returned k and q are differentiable in k_pe and q (reverse mode).  What
    enters the cache leaves the graph there: c_kv has no gradient from this call,
    and a cache or tables that require one are refused."""
    given = (cache, c_kv, k_pe, q, cos, sin)
    if _in_graph(*given) or _tangents(*given):
        return LatentAppend.apply(cache, c_kv, k_pe, slots, positions, cos, sin, q, interleaved, timer)
    return _append(cache, c_kv, k_pe, slots, positions, cos, sin, q, interleaved, timer)


class LatentAppend(torch.autograd.Function):
    """``append`` with the gradients of k_pe and q: a rotation is orthogonal, so
    they are the outputs' gradients turned back, by the angle's negative."""

    @staticmethod
    def forward(ctx, cache, c_kv, k_pe, slots, positions, cos, sin, q, interleaved, timer):
        if any(t is not None and t.requires_grad for t in (cache, cos, sin)):
            raise ValueError("latent append: cache, cos and sin have no gradient")
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, cos, sin)
        ctx.interleaved = interleaved
        ctx.k = k_pe.shape, k_pe.dtype, k_pe.device
        return _append(cache, c_kv, k_pe, slots, positions, cos, sin, q, interleaved, timer)

    @staticmethod
    @once_differentiable
    def backward(ctx, dk, dq):
        positions, cos, sin = ctx.saved_tensors
        shape, dtype, device = ctx.k
        k = torch.zeros(shape, dtype=dtype, device=device) if dk is None else dk.to(dtype)
        k, q = _append(None, None, k, None, positions, cos, -sin, None if dq is None else dq.to(dtype),
                       ctx.interleaved, None)
        return None, None, None if dk is None else k, None, None, None, None, q, None, None


def _append(cache, c_kv, k_pe, slots, positions, cos, sin, q, interleaved, timer):
    named = [("k_pe", k_pe)] + [(n, t) for n, t in (("c_kv", c_kv), ("cache", cache), ("q", q)) if t is not None]
    _operands("latent append", *named)
    if k_pe.dim() != 2:
        raise ValueError("latent append: k_pe must be [N, dr]")
    N, dr = k_pe.shape
    dev = k_pe.get_device()
    pages, page, dc, cs = 1, 1, 8, (0,)
    if cache is not None:
        if c_kv is None or slots is None or c_kv.dim() != 2 or c_kv.shape[0] != N:
            raise ValueError("latent append: c_kv must be [N, dc], with a slot for each token")
        dc = c_kv.shape[1]
        _cache("latent append", cache, dc + dr)
        pages, page = cache.shape[:2]
        slots = _index("latent append", "slots", slots, (N,), torch.int64, dev)
        c_kv, cs = _strided(c_kv, 1)
    positions = _index("latent append", "positions", positions, (N,), torch.int32, dev)
    cos, sin = _tables("latent append", cos, sin, dr, dev)
    k_pe, ks = _strided(k_pe, 1)
    H, dn, qs, q_out = 1, 8, (0, 0), None
    if q is not None:
        if q.dim() != 3 or q.shape[0] != N or q.shape[2] <= dr:
            raise ValueError("latent append: q must be [N, H, dn + dr]")
        q, qs = _strided(q, 2)
        H, dn = q.shape[1], q.shape[2] - dr
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(N, dr, dtype=k_pe.dtype, device=k_pe.device)
    if N == 0:
        return k_out, q_out
    args = _lib.LatentAppendArgs(N, H, dn, dr, dc, _DT[k_pe.dtype], page, pages, cos.shape[0], 1 if interleaved else 0,
                                 cs[0], ks[0], qs)
    if timer is not None:
        args.profile = timer.arm()
    rc = _lib.load().atomic_latent_append(ctypes.byref(args), _ptr(c_kv), _ptr(k_pe), _ptr(slots), _ptr(positions),
                                          _ptr(cos), _ptr(sin), _ptr(q), _ptr(cache), _ptr(k_out), _ptr(q_out),
                                          _stream(k_pe.device))
    _lib.check(rc, "atomic_latent_append")
    return k_out, q_out


def decode(q, w_kv, cache, page_table, kv_lens, scale, *, cos=None, sin=None, interleaved=False, workspace=None,
           timer=None):
    """o [B, n, H, dv]: n query tokens a sequence over its cached latents.

    ``q`` [B, n, H, dn + dr]; ``page_table`` int32 [B, pages of the longest];
    ``kv_lens`` int32 [B], the appended tokens counted in.  Query t of sequence
    b stands at position kv_lens[b] - n + t and sees the tokens up to and with
    its own; one before the sequence's start (as in an empty sequence) has
    o = 0.  With ``cos`` / ``sin`` the last dr elements of q are rotated by that
    position on the way, without them they are taken as rotated already.  An infinity
    or NaN in a cached row may reach the query tokens of the call that stand before it.

    The tokens are divided over the card by the table's width, not by the lengths (which
    the host does not know): hand over a table no wider than the longest sequence needs
    where it can be had (64 sequences of 1024 tokens, 16 heads: 42 us, with a table for
    131072 tokens 293).

    There is no gradient: in a graph (grad enabled and an input that requires it) a
    backward that comes back to o is an error, and forward-mode tangents are refused."""
    given = (q, w_kv, cache, cos, sin)
    if _in_graph(*given) or _tangents(*given):
        return LatentDecode.apply(q, w_kv, cache, page_table, kv_lens, scale, cos, sin, interleaved, workspace, timer)
    return _decode(q, w_kv, cache, page_table, kv_lens, scale, cos, sin, interleaved, workspace, timer)


class LatentDecode(torch.autograd.Function):
    """``decode`` in a graph, so that one which leads through it does not end there unnoticed."""

    @staticmethod
    def forward(ctx, *args):
        return _decode(*args)

    @staticmethod
    def backward(ctx, do):
        raise RuntimeError("latent decode has no gradient (latent.attention has one)")


def _decode(q, w_kv, cache, page_table, kv_lens, scale, cos, sin, interleaved, workspace, timer):
    _operands("latent decode", ("q", q), ("w_kv", w_kv), ("cache", cache))
    if q.dim() != 4 or w_kv.dim() != 3 or w_kv.shape[0] != q.shape[2]:
        raise ValueError("latent decode: q must be [B, n, H, dn + dr] and w_kv [H, dn + dv, dc]")
    B, n, H, d = q.shape
    dev = q.get_device()
    dc = w_kv.shape[2]
    if cache.dim() != 3 or not 0 < cache.shape[2] - dc < d or w_kv.shape[1] <= d - (cache.shape[2] - dc):
        raise ValueError("latent decode: cache must be [pages, page, dc + dr], w_kv [H, dn + dv, dc]")
    dr = cache.shape[2] - dc
    _cache("latent decode", cache, dc + dr)
    if page_table.dim() != 2:
        raise ValueError("latent decode: page_table must be int32 [B, pages]")
    page_table = _index("latent decode", "page_table", page_table, (B, page_table.shape[1]), torch.int32, dev)
    kv_lens = _index("latent decode", "kv_lens", kv_lens, (B,), torch.int32, dev)
    if (cos is None) != (sin is None):
        raise ValueError("latent decode: cos and sin come together")
    if cos is not None:
        cos, sin = _tables("latent decode", cos, sin, dr, dev)
    if not (q.numel() and page_table.numel()):      # no queries, or none with a token to see
        return q.new_zeros(B, n, H, w_kv.shape[1] - (d - dr))
    q, qs = _strided(q, 3)
    w_kv, _ = _strided(w_kv.contiguous(), 2)
    lib = _lib.load()
    args = _lib.LatentDecodeArgs(B, n, H, d - dr, dr, w_kv.shape[1] - (d - dr), dc, _DT[q.dtype], cache.shape[1],
                                 cache.shape[0], page_table.shape[1], 0 if cos is None else cos.shape[0],
                                 1 if interleaved else 0, scale, qs)
    if timer is not None:
        args.profile = timer.arm()
    nbytes = lib.atomic_latent_decode_workspace_size(ctypes.byref(args))
    if nbytes == 0:
        raise _lib.AtomicError("atomic_latent_decode_workspace_size: unsupported shape")
    workspace = _workspace(workspace, nbytes, q.device)
    o = torch.empty(B, n, H, args.dv, dtype=q.dtype, device=q.device)
    rc = lib.atomic_latent_decode(ctypes.byref(args), _ptr(q), _ptr(w_kv), _ptr(cache), _ptr(page_table),
                                  _ptr(kv_lens), _ptr(cos), _ptr(sin), _ptr(o), _ptr(workspace), workspace.numel(),
                                  _stream(q.device))
    _lib.check(rc, "atomic_latent_decode")
    return o

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
  ``append``         writes tokens into the cache and rotates keys and queries
  ``decode``         reads it; on request gathers each token's attention weight
  ``decode_shared``  the same for sequences that share a prefix, read once for all
  ``evict``          leaves the tokens with the largest weights in the cache
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
    """The current stream's handle.  (As torch.cuda.current_stream gives it, without the 1.7 us of a Stream object.)"""
    return torch._C._cuda_getCurrentRawStream(device.index)


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
    if q.get_device() != torch.cuda.current_device():      # the library launches on the current device
        with torch.cuda.device(q.device):
            return forward(q, kv, k_pe, scale, causal=causal, q_lens=q_lens, kv_lens=kv_lens, save=save,
                           workspace=workspace, timer=timer)
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
    if q.get_device() != torch.cuda.current_device():      # the library launches on the current device
        with torch.cuda.device(q.device):
            return backward(q, kv, k_pe, o, lse, dout, scale, causal=causal, q_lens=q_lens, kv_lens=kv_lens, rest=rest,
                            workspace=workspace, timer=timer)
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
    if k_pe.get_device() != torch.cuda.current_device():      # the library launches on the current device
        with torch.cuda.device(k_pe.device):
            return _append(cache, c_kv, k_pe, slots, positions, cos, sin, q, interleaved, timer)
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


def decode(q, w_kv, cache, page_table, kv_lens, scale, *, cos=None, sin=None, interleaved=False, weights=None,
           workspace=None, timer=None):
    """o [B, n, H, dv]: n query tokens a sequence over its cached latents.

    ``q`` [B, n, H, dn + dr]; ``page_table`` int32 [B, pages of the longest];
    ``kv_lens`` int32 [B], the appended tokens counted in.  Query t of sequence
    b stands at position kv_lens[b] - n + t and sees the tokens up to and with
    its own; one before the sequence's start (as in an empty sequence) has
    o = 0.  With ``cos`` / ``sin`` the last dr elements of q are rotated by that
    position on the way, without them they are taken as rotated already (by
    ``append``, as after an eviction, when the rows say nothing of the positions).
    An infinity or NaN in a cached row may reach the query tokens of the call that
    stand before it.

    ``weights`` float32 [B, tokens of the table or more] gathers what ``evict`` goes by:
    to weights[b, j] is added, in place, the sum over heads and query tokens of the
    softmax weight of token j; those of the n newest tokens are set to it, they begin
    here.  What lies past the length stays as it is.  The query then enters the scores
    as two bfloat16 numbers, so that the weights are float32's (and o a little nearer
    to the exact one than without them).

    The tokens are divided over the card by the table's width, not by the lengths (which
    the host does not know): hand over a table no wider than the longest sequence needs
    where it can be had (64 sequences of 1024 tokens, 16 heads: 42 us, with a table for
    131072 tokens 293).

    There is no gradient: in a graph (grad enabled and an input that requires it) a
    backward that comes back to o is an error, and forward-mode tangents are refused."""
    given = (q, w_kv, cache, cos, sin, weights)
    args = (q, w_kv, cache, None, None, page_table, kv_lens, scale, cos, sin, interleaved, weights, workspace, timer)
    return (LatentDecode.apply if _in_graph(*given) or _tangents(*given) else _decode)(*args)


def decode_shared(q, w_kv, cache, prefix_table, prefix_lens, page_table, kv_lens, scale, *, cos=None, sin=None,
                  interleaved=False, weights=None, workspace=None, timer=None):
    """``decode`` for sequences that share prefixes, each read once for all that follow it.

    ``prefix_table`` int32 [G, pages of the longest] and ``prefix_lens`` int32 [G]
    are the prefixes' tokens in the same cache; the batch is G equal runs, sequence b
    follows prefix b // (B / G).  ``page_table`` and ``kv_lens`` are each sequence's own
    tokens, those after the prefix (a length of zero: the prefix only).  Query t
    stands at position prefix_lens[g] + kv_lens[b] - n + t and sees the tokens up to and
    with its own: what ``decode`` gives for the two tables as one, up to rounding.
    ``weights`` are those of the own tokens; a prefix's are not gathered.

    In bfloat16, with more than 32 query rows (tokens and heads) behind a prefix whose
    table holds 4096 tokens or more, what the prefix adds is rounded otherwise than in
    ``decode``: a probability enters as one bfloat16 number from a prefix length of 2048
    on (o is off by 0.0025 of its norm where decode's is by 0.0023), and with ``weights``
    the query's second number enters o's scores in its rotated part only, the weights by
    its first order (they are off by 1.5e-6 of their norm at scores of unit spread, by
    2e-5 to 3e-5 at a spread of 10; decode's by 1e-6 and 8e-6).

    Both tables' widths divide the tokens over the card, as in ``decode`` (64 sequences of
    16 heads, 8192 prefix and 1024 own tokens: 66 us, with a prefix table for 32768 tokens
    104, with own tables for 8192 128), and an idle sequence that fills a run up costs its
    rows' share of the prefix."""
    if (prefix_table is None) != (prefix_lens is None):
        raise ValueError("latent decode: prefix_table and prefix_lens come together")
    given = (q, w_kv, cache, cos, sin, weights)
    args = (q, w_kv, cache, prefix_table, prefix_lens, page_table, kv_lens, scale, cos, sin, interleaved, weights,
            workspace, timer)
    return (LatentDecode.apply if _in_graph(*given) or _tangents(*given) else _decode)(*args)


class LatentDecode(torch.autograd.Function):
    """``decode`` in a graph, so that one which leads through it does not end there unnoticed."""

    @staticmethod
    def forward(ctx, *args):
        return _decode(*args)

    @staticmethod
    def backward(ctx, do):
        raise RuntimeError("latent decode has no gradient (latent.attention has one)")


def _per_token(what, name, t, B, least, dtype, device):
    """Checks a [B, tokens] state whose rows the library reads or writes in place; its row stride."""
    if t.dtype != dtype or t.dim() != 2 or t.shape[0] != B or not least <= t.shape[1] < 1 << 31 or \
            t.get_device() != device or t.requires_grad:
        raise ValueError(f"{what}: {name} must be {str(dtype)[6:]} [{B}, {least} or more] on the inputs' device, "
                         "without a gradient")
    if t.shape[1] > 1 and t.stride(1) != 1 or B > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: {name} must have dense rows that do not overlap")
    return t.stride(0) if B > 1 else t.shape[1]


def _decode(q, w_kv, cache, prefix_table, prefix_lens, page_table, kv_lens, scale, cos, sin, interleaved, weights,
            workspace, timer):
    _operands("latent decode", ("q", q), ("w_kv", w_kv), ("cache", cache))
    if q.get_device() != torch.cuda.current_device():      # the library launches on the current device
        with torch.cuda.device(q.device):
            return _decode(q, w_kv, cache, prefix_table, prefix_lens, page_table, kv_lens, scale, cos, sin, interleaved,
                           weights, workspace, timer)
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
    G = front = 0
    if prefix_table is not None:
        if prefix_table.dim() != 2 or prefix_lens.dim() != 1:
            raise ValueError("latent decode: prefix_table must be int32 [G, pages] and prefix_lens int32 [G]")
        G, front = prefix_table.shape
        if G == 0 and B or G and B % G:
            raise ValueError(f"latent decode: {G} prefixes do not divide a batch of {B}")
        prefix_table = _index("latent decode", "prefix_table", prefix_table, (G, front), torch.int32, dev)
        prefix_lens = _index("latent decode", "prefix_lens", prefix_lens, (G,), torch.int32, dev)
    if (cos is None) != (sin is None):
        raise ValueError("latent decode: cos and sin come together")
    if cos is not None:
        cos, sin = _tables("latent decode", cos, sin, dr, dev)
    stride = 0
    if weights is not None:
        stride = _per_token("latent decode", "weights", weights, B, page_table.shape[1] * cache.shape[1], torch.float32,
                            dev)
    if not (q.numel() and (page_table.numel() or front)):      # no queries, or none with a token to see
        return q.new_zeros(B, n, H, w_kv.shape[1] - (d - dr))
    q, qs = _strided(q, 3)
    w_kv, _ = _strided(w_kv.contiguous(), 2)
    lib = _lib.load()
    args = _lib.LatentDecodeArgs(B, n, H, d - dr, dr, w_kv.shape[1] - (d - dr), dc, _DT[q.dtype], cache.shape[1],
                                 cache.shape[0], page_table.shape[1], 0 if cos is None else cos.shape[0],
                                 1 if interleaved else 0, scale, qs)
    if timer is not None:
        args.profile = timer.arm()
    plain = not G and weights is None
    if not plain:
        args = _lib.LatentSharedArgs(args, G, front, weights is not None, stride)
    size = lib.atomic_latent_decode_workspace_size if plain else lib.atomic_latent_decode_shared_workspace_size
    nbytes = size(ctypes.byref(args))
    if nbytes == 0:
        raise _lib.AtomicError("atomic_latent_decode_workspace_size: unsupported shape")
    workspace = _workspace(workspace, nbytes, q.device)
    o = torch.empty(B, n, H, w_kv.shape[1] - (d - dr), dtype=q.dtype, device=q.device)
    if plain:
        rc = lib.atomic_latent_decode(ctypes.byref(args), _ptr(q), _ptr(w_kv), _ptr(cache), _ptr(page_table),
                                      _ptr(kv_lens), _ptr(cos), _ptr(sin), _ptr(o), _ptr(workspace),
                                      workspace.numel(), _stream(q.device))
        _lib.check(rc, "atomic_latent_decode")
    else:
        rc = lib.atomic_latent_decode_shared(ctypes.byref(args), _ptr(q), _ptr(w_kv), _ptr(cache), _ptr(prefix_table),
                                             _ptr(prefix_lens), _ptr(page_table), _ptr(kv_lens), _ptr(cos), _ptr(sin),
                                             _ptr(weights), _ptr(o), _ptr(workspace), workspace.numel(),
                                             _stream(q.device))
        _lib.check(rc, "atomic_latent_decode_shared")
    return o


def evict(cache, page_table, kv_lens, weights, order, keep, *, sinks=0, recent=1, in_place=False, workspace=None,
          timer=None):
    """``(kv_lens, weights, order, source)`` after an eviction: of each sequence with
    more than ``keep`` tokens, keep stay in the cache.

    ``weights`` float32 [B, W] are the tokens' gathered attention weights (``decode``)
    and ``order`` int32 [B, W] their places among all tokens of their sequence, W being
    the table's tokens or more.  order holds -1 in rows that no eviction has seen: such
    tokens are taken as the newest, in the order of their rows, so a program begins
    with -1 everywhere and hands on what this call returns.  The first ``sinks`` tokens
    (order < sinks) and those of the ``recent`` last places (order above the newest one's
    less recent; a place whose token an earlier call with a smaller recent evicted
    stays empty) are kept whatever their weights, of the others
    those with the largest (equal ones: the lowest rows first; a NaN counts as the
    least).  Kept tokens in rows past keep move into the rows below that became free, in
    the order of the rows on both sides; nothing else in ``cache`` is written.

    The new kv_lens are at most keep; the new weights and order hold 0 and -1 past
    them.  ``source`` int32 [B, keep] is the row that each row's token was in (-1 past
    the length).  With ``in_place`` kv_lens, weights and order are written over and
    returned.  Without it the inputs stay, and the same call does the same once more.
    A sequence's pages must be its own: of a prefix that others share, only what
    follows it can be evicted (``decode_shared``)."""
    what = "latent evict"
    if not cache.is_cuda:
        raise ValueError(f"{what}: inputs must be HIP device tensors")
    if cache.dtype not in _DT:
        raise TypeError(f"{what}: cache must be bfloat16 or float32")
    if cache.get_device() != torch.cuda.current_device():      # the library launches on the current device
        with torch.cuda.device(cache.device):
            return evict(cache, page_table, kv_lens, weights, order, keep, sinks=sinks, recent=recent, in_place=in_place,
                         workspace=workspace, timer=timer)
    if cache.dim() != 3 or cache.requires_grad:
        raise ValueError(f"{what}: cache must be a dense [pages, page, dc + dr], without a gradient")
    if _tangents(cache, weights):
        raise NotImplementedError(f"{what}: no tangents in forward mode: cache and weights must have none")
    _cache(what, cache, cache.shape[2])
    dev = cache.get_device()
    if page_table.dim() != 2:
        raise ValueError(f"{what}: page_table must be int32 [B, pages]")
    B, per = page_table.shape
    page_table = _index(what, "page_table", page_table, (B, per), torch.int32, dev)
    lens = _index(what, "kv_lens", kv_lens, (B,), torch.int32, dev)
    if in_place and lens is not kv_lens:
        raise ValueError(f"{what}: kv_lens must be dense to be written in place")
    if not 1 <= keep <= 1 << 30 or not 0 <= sinks <= keep or not 0 <= recent <= keep - sinks:
        raise ValueError(f"{what}: keep must be 1 .. 2^30, sinks and recent 0 or more and together at most keep")
    pages, page, row = cache.shape
    ws = _per_token(what, "weights", weights, B, per * page, torch.float32, dev)
    os = _per_token(what, "order", order, B, per * page, torch.int32, dev)
    if order.shape != weights.shape:
        raise ValueError(f"{what}: weights and order must have one shape")
    W = weights.shape[1]
    source = torch.empty(B, keep, dtype=torch.int32, device=cache.device)
    if in_place:
        out, wos, oos = (kv_lens, weights, order), ws, os
    else:
        out, wos, oos = (torch.empty_like(lens), weights.new_empty(B, W), order.new_empty(B, W)), W, W
    if not (B and per and pages and page):      # no token anywhere
        out[0].zero_(), out[1].zero_(), out[2].fill_(-1), source.fill_(-1)
        return (*out, source)
    lib = _lib.load()
    args = _lib.LatentEvictArgs(B, _DT[cache.dtype], row, page, pages, per, W, keep, sinks, recent, ws, os, wos, oos)
    if timer is not None:
        args.profile = timer.arm()
    nbytes = lib.atomic_latent_evict_workspace_size(ctypes.byref(args))
    if nbytes == 0:
        raise _lib.AtomicError("atomic_latent_evict: ATOMIC_ERR_SHAPE: unsupported or inconsistent dimensions",
                               _lib.ATOMIC_ERR_SHAPE)
    workspace = _workspace(workspace, nbytes, cache.device)
    rc = lib.atomic_latent_evict(ctypes.byref(args), _ptr(cache), _ptr(page_table), _ptr(lens), _ptr(weights),
                                 _ptr(order), *(_ptr(t) for t in out), _ptr(source), _ptr(workspace),
                                 workspace.numel(), _stream(cache.device))
    _lib.check(rc, "atomic_latent_evict")
    return (*out, source)

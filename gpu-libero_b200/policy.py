"""Operators of a learned policy that acts in, and learns from, the batched worlds.

A policy reads one observation row per world and control step
(`Runtime.buffers['obs']`), keeps a memory per world, and writes the worlds'
actions, all on the device that steps them:

- `decay_attention_step`: linear attention with a decay for each head, one
  token per world: the recurrent form, used while acting;
- `decay_attention`: the same over trajectories, with its gradients: used to
  read a recorded prefix and to learn from rollouts;
- `layer_norm`: with its gradients;
- `clip_grad_norm`: the global gradient norm over many tensors, and clipping.

Every operator runs on hand-written kernels of libb200policy.so on the current
stream of its tensors' device, allocates through PyTorch's allocator, and
does not wait for the device (`check` does, and so does a device's first call).
There is no CPU fallback: tensors that are not on a CUDA device are refused.
Types are float32, float16 and bfloat16; states, statistics and sums are float32
or wider.  Arguments that do not fit raise ValueError before any device work.

What trajectories round to fewer bits: their products run on tensor cores, which
take the weights q . k of a token's keys, and the copy of the state that a chunk of
tokens reads, in 8 bits for bfloat16, in 11 for float16 and in two terms of 11 for float32.  An
output or gradient of 16 bits is off by 1.4 times what its own rounding takes (root
mean square: 0.0023 of its size in bfloat16, 0.00029 in float16), one of float32 by
5e-7.  The states that a trajectory leaves have 32 bits, and acting reads the 32-bit
state itself, so that the same tokens give slightly different outputs in the two.
"""
import math
import struct

import torch
from torch.autograd import forward_ad

from . import native

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
HEAD_MAX = 128  # B200_HEAD_MAX of include/b200policy.h
INDEX_MAX = (1 << 31) - 1 - 1024  # tokens of a row, and columns of a norm: the kernels count them in 32 bits
ATTENTION_WORKSPACE, NORM_WORKSPACE = 15 * 8, 9 * 8  # offsets of the structs' workspace fields

_library = None


def _lib():
    global _library
    if _library is None:
        _library = native.PolicyLibrary()
    return _library


# The current stream's handle; the public call makes a Stream object (2 us a call).
_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _launch(device, name, *args):
    """One library call on the current stream of `device`, made current if it is not."""
    index = device.index
    if index == torch.cuda.current_device():
        _lib().launch(name, *args, _stream(index))
    else:
        with torch.cuda.device(device):
            _lib().launch(name, *args, _stream(index))


# Kernels write through pointers: raising the version of the tensors that they wrote lets
# autograd refuse a backward pass that has saved one of them, as for PyTorch's own in-place calls.
_wrote = torch.autograd.graph.increment_version

_status_words = {}


def _status(device):
    """The address of the device's status word.

    Zero if it would have to be made during a capture: such a call takes kernels that need none."""
    word = _status_words.get(device)
    if word is None:
        if device.type != 'cuda' or torch.cuda.is_current_stream_capturing():
            return 0
        with torch.inference_mode(False):  # check() clears it in any mode
            word = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()  # once: any stream may read it from now on
        _status_words[device] = word
    return word.data_ptr()


def check(device='cuda'):
    """Raise if a kernel's bounded wait has run out on `device` since the last check.

    The outputs of the call that it ran out in are void; which call that was is not known.  Later calls
    are not affected, except replays of a CUDA graph that holds that call: theirs are void until this
    check.  Waits for the device; the operators themselves never do."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    torch.cuda.synchronize(device)
    word = _status_words.get(device)
    if word is not None and int(word.item()):
        word.zero_()
        torch.cuda.synchronize(device)
        raise RuntimeError('a decay attention kernel gave up waiting on %s since the last check; the outputs of its call '
                           'are void' % device)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _require(condition, message, *values):
    if not condition:
        raise ValueError(message % values if values else message)


def _forward_mode():
    """Whether this is inside a dual level: no tensor has a tangent elsewhere."""
    return getattr(forward_ad, '_current_level', 0) >= 0


def _refuse_tangents(*tensors):
    """Forward-mode derivatives are refused: the kernels would drop them without a word."""
    for t in tensors if _forward_mode() else ():
        _require(not isinstance(t, torch.Tensor) or forward_ad.unpack_dual(t).tangent is None,
                 'the policy operators have no forward-mode derivatives')


def _rows(t):
    """`t`, or a copy whose last dimension is contiguous."""
    return t if t.is_contiguous() or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _once(backward):
    """A Function's backward that only takes the detour of refusing second
    derivatives where a graph of the backward pass is asked for."""
    strict = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return strict(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return staticmethod(run)


# ---- decay attention -------------------------------------------------------
def _explain_attention(q, k, v, log_decay, state, first, lengths, lead):
    """Raise for the first argument of a call that does not fit."""
    rank = len(lead) + 2
    _require(q.dtype in DTYPES, 'q must be float32, float16 or bfloat16, not %s', q.dtype)
    _require(q.dim() == rank and k.dim() == rank and v.dim() == rank, 'q, k and v must be [%s, heads, width]',
             ', '.join(lead))
    _require(k.dtype == q.dtype and v.dtype == q.dtype, 'q, k and v must have one type')
    device = q.device
    for name, t in (('k', k), ('v', v), ('log_decay', log_decay), ('state', state), ('first', first),
                    ('lengths', lengths)):
        _require(t is None or t.device == device, '%s must be on %s', name, device)
    at = q.shape[:-2]
    heads, dk = q.shape[-2:]
    kv_heads, dv = v.shape[-2:]
    _require(k.shape[:-2] == at and v.shape[:-2] == at and k.shape[-2] == kv_heads and k.shape[-1] == dk,
             'q %s, k %s and v %s do not fit together', tuple(q.shape), tuple(k.shape), tuple(v.shape))
    _require(kv_heads > 0 and heads > 0 and heads % kv_heads == 0,
             '%d query heads cannot share %d key and value heads', heads, kv_heads)
    _require(0 < dk <= HEAD_MAX and 0 < dv <= HEAD_MAX, 'head widths must be 1 to %d, not %d and %d', HEAD_MAX, dk, dv)
    _require(log_decay.shape == (heads,) and log_decay.dtype == torch.float32,
             'log_decay must be float32 of shape (%d,)', heads)
    _require(not (log_decay.requires_grad and torch.is_grad_enabled()),
             'log_decay is a constant of the heads: it has no gradient')
    _require(state is None or (state.shape == (at[0], heads, dk, dv) and state.dtype == torch.float32),
             'state must be float32 of shape %s', (at[0], heads, dk, dv))
    _require(first is None or (first.shape == at and first.dtype == torch.bool), 'first must be bool of shape %s',
             tuple(at))
    _require(lengths is None or (lengths.shape == at[:1] and lengths.dtype == torch.int32),
             'lengths must be int32 of shape (%d,)', at[0])
    _require(at[0] * heads < 1 << 31, 'too many rows: %d', at[0] * heads)
    _require(len(at) == 1 or at[1] <= INDEX_MAX, 'too many tokens: %d', at[-1])
    _require(q.is_cuda, 'decay attention needs CUDA tensors')


def _check_attention(q, k, v, log_decay, state, first, lengths, scale, lead):
    """The scale of a call whose arguments fit; `lead` names the dimensions before the heads."""
    dtype, device, at = q.dtype, q.device, q.shape[:-2]
    fits = dtype in DTYPES and q.is_cuda and q.dim() == len(lead) + 2
    if fits:
        (heads, dk), (kv_heads, dv) = q.shape[-2:], v.shape[-2:]
        fits = (k.dtype is dtype and v.dtype is dtype and k.shape == (*at, kv_heads, dk) and v.shape[:-2] == at
                and kv_heads and heads and not heads % kv_heads and 0 < dk <= HEAD_MAX and 0 < dv <= HEAD_MAX
                and k.device == device and v.device == device and log_decay.device == device
                and log_decay.dtype is torch.float32 and log_decay.shape == (heads,)
                and not (log_decay.requires_grad and torch.is_grad_enabled()) and at[0] * heads < 1 << 31
                and (len(at) == 1 or at[1] <= INDEX_MAX)
                and (state is None or (state.shape == (at[0], heads, dk, dv) and state.dtype is torch.float32
                                       and state.device == device))
                and (first is None or (first.shape == at and first.dtype is torch.bool and first.device == device))
                and (lengths is None or (lengths.shape == at[:1] and lengths.dtype is torch.int32
                                         and lengths.device == device)))
    if not fits:
        _explain_attention(q, k, v, log_decay, state, first, lengths, lead)
        raise ValueError('decay attention: arguments do not fit')
    return dk ** -0.5 if scale is None else float(scale)


def _pack(q, k, v, log_decay, state, first, lengths, scale, out, state_out, dout, dstate_out, dq, dk, dv, dstate):
    """The B200AttentionArgs of one launch, as bytes; its workspace is to be set."""
    at, qs, ks, vs = native.PolicyLibrary.ATTENTION.pack, q.stride(), k.stride(), v.stride()
    if len(qs) == 3:  # one token: a time axis of length one
        strides = (qs[0], 0, qs[1], ks[0], 0, ks[1], vs[0], 0, vs[1], 0, 0, 0, 0 if first is None else first.stride(0), 0)
        batch, heads, width = q.shape
        time = 1
    else:
        strides = (*qs[:3], *ks[:3], *vs[:3], *((0, 0, 0) if dout is None else dout.stride()[:3]),
                   *((0, 0) if first is None else first.stride()))
        batch, time, heads, width = q.shape
    return at(q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), _ptr(state), _ptr(first), _ptr(lengths),
              _ptr(out), _ptr(state_out), _ptr(dout), _ptr(dstate_out), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dstate), 0,
              _status(q.device),
              *strides, batch, time, heads, v.shape[-2], width, v.shape[-1], DTYPES[q.dtype], scale)


def _with_workspace(name, args, place, device, *more):
    """`args` with the workspace that the library asks for at byte `place`, and that tensor."""
    size = _lib().size(name, args, *more)
    if not size:
        return args, None
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    return args[:place] + workspace.data_ptr().to_bytes(8, 'little') + args[place + 8:], workspace


def _attention_forward(q, k, v, log_decay, state, first, lengths, scale, state_out=None):
    out = q.new_empty(q.shape[:-1] + v.shape[-1:])
    if state_out is None:
        state_out = log_decay.new_empty((q.shape[0], q.shape[-2], q.shape[-1], v.shape[-1]))
    args = _pack(q, k, v, log_decay, state, first, lengths, scale, out, state_out, None, None, None, None, None, None)
    workspace = None
    if q.dim() == 4:
        args, workspace = _with_workspace('attention', args, ATTENTION_WORKSPACE, q.device, 0)
    _launch(q.device, 'attention_forward', args)
    return out, state_out


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, first, lengths, scale):
        out, state_out = _attention_forward(q, k, v, log_decay, state, first, lengths, scale)
        ctx.save_for_backward(q, k, v, log_decay, state, first, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, state_out

    @_once
    def backward(ctx, dout, dstate_out):
        q, k, v, log_decay, state, first, lengths = ctx.saved_tensors
        if dout is None:
            dout = q.new_zeros(()).expand(q.shape[:-1] + v.shape[-1:])
        dout = _rows(dout)
        if dstate_out is not None:
            dstate_out = dstate_out.contiguous()
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        dstate = state.new_empty(state.shape) if state is not None and ctx.needs_input_grad[4] else None
        args = _pack(q, k, v, log_decay, state, first, lengths, ctx.scale, None, None, dout, dstate_out, dq, dk, dv,
                     dstate)
        args, workspace = _with_workspace('attention', args, ATTENTION_WORKSPACE, q.device, 1)
        _launch(q.device, 'attention_backward', args)
        return dq, dk, dv, None, dstate, None, None, None


def decay_attention(q, k, v, log_decay, *, scale=None, state=None, first=None, lengths=None):
    """Linear attention with a decay for each head, over trajectories.

    For each world b and head h, with lambda = exp(log_decay[h]):

        S_t = lambda * (0 if first[b, t] else S_{t-1}) + k_t v_t^T
        o_t = scale * q_t S_t

    Arguments
    - q [batch, time, heads, dk]; k [batch, time, kv_heads, dk]; v [batch,
      time, kv_heads, dv]: one type, any strides (a last dimension that is not
      contiguous is copied).  heads is a multiple of kv_heads: query head h
      reads key / value head h // (heads // kv_heads).  dk and dv: 1 to 128.
    - log_decay [heads], float32, at most zero (-inf: no memory).  A constant.
    - scale: dk ** -0.5 by default.
    - state [batch, heads, dk, dv], float32: the memory before the first token
      (None: zero).
    - first [batch, time], bool: the token starts an episode; the memory is
      cleared before it.
    - lengths [batch], int32: row b holds lengths[b] tokens; what q, k and v
      hold behind them is never used, and their output and gradients are zero.

    Returns (out [batch, time, heads, dv] in q's type, state [batch, heads, dk,
    dv] in float32 after each row's last token).  Differentiable in q, k, v
    and state, once (not in forward mode).  Tokens of a row must be finite;
    those behind its length may hold anything.
    """
    _refuse_tangents(q, k, v, log_decay, state)
    scale = _check_attention(q, k, v, log_decay, state, first, lengths, scale, ('batch', 'time'))
    q, k, v = _rows(q), _rows(k), _rows(v)
    log_decay = log_decay.contiguous()
    state = None if state is None else state.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (state is not None and state.requires_grad)):
        return _DecayAttention.apply(q, k, v, log_decay, state, first, lengths, scale)
    return _attention_forward(q, k, v, log_decay, state, first, lengths, scale)


def decay_attention_step(q, k, v, log_decay, state, *, scale=None, first=None, state_out=None):
    """One token of `decay_attention` for every world: the recurrent form.

    q [batch, heads, dk], k [batch, kv_heads, dk], v [batch, kv_heads, dv],
    first [batch]; log_decay, scale and state as there.  The new memory goes to
    `state_out` (dense float32 like state; `state` itself for an update in
    place; it may share memory with no other argument), or to a new tensor.  Returns (out [batch, heads, dv], new state).
    An update in place counts as one for autograd: a backward pass that has
    saved the old memory is refused.
    Acting keeps no graph: arguments that require gradients are refused.
    """
    _require(state is not None, 'decay_attention_step needs a state')
    _refuse_tangents(q, k, v, log_decay, state, state_out)
    scale = _check_attention(q, k, v, log_decay, state, first, None, scale, ('batch',))
    if torch.is_grad_enabled():
        _require(not (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad),
                 'decay_attention_step keeps no graph: use decay_attention, or torch.no_grad()')
    if state_out is not None:
        _require(state_out.shape == state.shape and state_out.dtype == torch.float32 and state_out.is_contiguous()
                 and state_out.device == q.device, 'state_out must be dense float32 of shape %s on %s',
                 tuple(state.shape), q.device)
        _require(not (state_out.requires_grad and torch.is_grad_enabled()), 'state_out must not require gradients')
        if state_out is not state and state.is_contiguous():  # (one that is not is read from a dense copy)
            apart = abs(state_out.data_ptr() - state.data_ptr())
            _require(apart == 0 or apart >= 4 * state.numel(), 'state_out must be state itself or share no memory with it')
    result = _attention_forward(_rows(q), _rows(k), _rows(v), log_decay.contiguous(), state.contiguous(), first, None,
                                scale, state_out)
    if state_out is not None:
        _wrote(state_out)
    return result


# ---- layer norm ------------------------------------------------------------
def _norm_pack(x, weight, bias, eps, y, stats, dy, dx, dweight, dbias):
    """The B200NormArgs of one launch, as bytes, its workspace to be set; x and dy are [rows, width]."""
    typed = x if weight is None and bias is None else bias if weight is None else weight
    return native.PolicyLibrary.NORM.pack(
        x.data_ptr(), _ptr(weight), _ptr(bias), _ptr(y), _ptr(stats), _ptr(dy), _ptr(dx), _ptr(dweight), _ptr(dbias),
        0, x.shape[0], x.stride(0), 0 if dy is None else dy.stride(0), x.shape[1], DTYPES[x.dtype],
        DTYPES[typed.dtype], eps)


def _as_rows(t):
    """`t` as [rows, width] with a contiguous width: a view where one exists."""
    return _rows(t if t.dim() == 2 else t.reshape(-1, t.shape[-1]))


def _norm_forward(x, weight, bias, eps, keep):
    flat = _as_rows(x)
    y = x.new_empty(x.shape)
    stats = x.new_empty((flat.shape[0], 2), dtype=torch.float32) if keep else None
    _launch(x.device, 'norm_forward', _norm_pack(flat, weight, bias, eps, y, stats, None, None, None, None))
    return y, flat, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, flat, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(flat, weight, bias, stats)
        ctx.eps, ctx.shape = eps, x.shape
        return y

    @_once
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = x.new_empty(ctx.shape) if need[0] else None
        dweight = weight.new_empty(weight.shape) if need[1] else None
        dbias = bias.new_empty(bias.shape) if need[2] else None
        args = _norm_pack(x, weight, bias, ctx.eps, None, stats, _as_rows(dy), dx, dweight, dbias)
        workspace = None
        if dweight is not None or dbias is not None:
            args, workspace = _with_workspace('norm', args, NORM_WORKSPACE, x.device)
        _launch(x.device, 'norm_backward', args)
        return dx, dweight, dbias, None


def _explain_norm(x, weight, bias, eps):
    """Raise for the first argument of a call that does not fit."""
    _require(x.dtype in DTYPES, 'x must be float32, float16 or bfloat16, not %s', x.dtype)
    _require(x.dim() >= 1 and x.shape[-1] > 0, 'layer_norm needs a last dimension, not shape %s', tuple(x.shape))
    for name, t in (('weight', weight), ('bias', bias)):
        _require(t is None or (t.shape == x.shape[-1:] and t.dtype in (x.dtype, torch.float32)
                               and t.device == x.device), '%s must have shape (%d,) and type %s or float32, on %s',
                 name, x.shape[-1], x.dtype, x.device)
    _require(weight is None or bias is None or weight.dtype == bias.dtype, 'weight and bias must have one type')
    _require(eps >= 0 and math.isfinite(eps), 'eps must be finite and not negative')
    _require(x.numel() // x.shape[-1] < 1 << 31, 'too many rows')
    _require(x.shape[-1] <= INDEX_MAX, 'too many columns: %d', x.shape[-1])
    _require(x.is_cuda, 'layer_norm needs a CUDA tensor')


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x [..., width]; rows may be strided (a slice of a wider observation slab).
    weight and bias [width]: x's type or float32, both the same, or None.
    Returns a dense tensor of x's shape and type.  Mean, variance and the sums
    of the gradients are held in float32.  Differentiable in x, weight and
    bias, once (not in forward mode); gradients of weight and bias are summed in
    a fixed order.
    """
    _refuse_tangents(x, weight, bias)
    dtype, width, eps = x.dtype, x.shape[-1] if x.dim() else 0, float(eps)
    if not (dtype in DTYPES and 0 < width <= INDEX_MAX and x.is_cuda and 0 <= eps < math.inf
            and (weight is None or (weight.shape == (width,) and weight.device == x.device
                                    and (weight.dtype is dtype or weight.dtype is torch.float32)))
            and (bias is None or (bias.shape == (width,) and bias.device == x.device
                                  and (bias.dtype is dtype or bias.dtype is torch.float32)))
            and (weight is None or bias is None or weight.dtype is bias.dtype) and x.numel() // width < 1 << 31):
        _explain_norm(x, weight, bias, eps)
        raise ValueError('layer_norm: arguments do not fit')
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


# ---- gradient clipping -----------------------------------------------------
def _dense(t):
    """Whether t's elements fill one stretch of memory, each once."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size != 1:
            if stride != expected:
                return False
            expected *= size
    return True


def _same_order(a, b):
    """Whether two tensors of one shape lay their elements out alike (strides of single elements do not count)."""
    return not a.numel() or all(n == 1 or i == j for n, i, j in zip(a.shape, a.stride(), b.stride()))


def _explain_overlap(entries):
    """Raise if memory that a clipping call writes belongs to two of its tensors."""
    ranges = []
    for src, dst, count, dtype in zip(*[iter(entries)] * 4):
        size = count * (4 if dtype == DTYPES[torch.float32] else 2)
        if size:
            ranges.append((dst, dst + size, True))
            if src != dst:
                ranges.append((src, src + size, False))
    written = taken = 0
    for low, high, write in sorted(ranges):
        _require(low >= (taken if write else written), 'gradients (and out) must not share memory: a value would be '
                 'scaled more than once')
        taken = max(taken, high)
        written = max(written, high) if write else written


def clip_grad_norm(grads, max_norm, *, eps=1e-6, out=None):
    """Scale gradients so that their global norm is at most `max_norm`.

        norm = sqrt(sum over all tensors of |g|^2)
        g <- g * min(1, max_norm / (norm + eps))

    grads: CUDA tensors of one device, of any mix of float32, float16 and
    bfloat16 and any shapes whose memory is dense; None is skipped.  They are
    scaled in place, or into the tensors of `out` (None where grads has None;
    same shapes, types and strides).  What is written may not share memory with
    another tensor of the call: a gradient that is listed twice in place, or an
    `out` that overlaps a gradient other than its own, is refused.  Returns the norm before clipping, a
    float32 scalar tensor on the device: nothing waits for it.  The sum of the
    squares is held in 64 bits and its order is fixed.  An infinite norm
    scales to zero (infinities to NaN) and a norm that is not a number makes
    every gradient so, as the formula says.
    """
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    to = grads if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
    if _forward_mode():
        _refuse_tangents(*grads, *to)
    _require(len(to) == len(grads), 'out has %d tensors for %d gradients', len(to), len(grads))
    max_norm, eps = float(max_norm), float(eps)
    _require(max_norm >= 0 and eps >= 0, 'max_norm and eps must not be negative')
    table, device = [], None
    for g, d in zip(grads, to):
        if g is None:
            _require(d is None, 'out has a tensor where there is no gradient')
            continue
        dtype = g.dtype
        if device is None:
            device = g.device
        if not (dtype in DTYPES and g.device == device and (g.is_contiguous() or (g.layout is torch.strided and _dense(g)))):
            _require(g.device == device, 'gradients must be on one device')
            _require(dtype in DTYPES and g.layout is torch.strided,
                     'gradients must be dense float32, float16 or bfloat16, not %s', dtype)
            raise ValueError('gradients must fill their memory densely: shape %s, strides %s'
                             % (tuple(g.shape), g.stride()))
        if d is not g and (d is None or d.shape != g.shape or d.dtype is not dtype or d.device != device
                           or (d.stride() != g.stride() and not _same_order(g, d))):
            raise ValueError('out must match its gradient in shape, type, strides and device')
        table += (g.data_ptr(), d.data_ptr(), g.numel(), DTYPES[dtype])
    if device is None:
        raise ValueError('clip_grad_norm needs at least one gradient')
    if device.type != 'cuda':
        _explain_overlap(table)
        raise ValueError('clip_grad_norm needs CUDA tensors')
    count = len(table) // 4
    entries, table = table, struct.pack('=%dq' % len(table), *table)
    norm = torch.empty((), dtype=torch.float32, device=device)
    workspace = torch.empty(_lib().size('clip', table, count), dtype=torch.uint8, device=device)
    try:
        _launch(device, 'clip', table, count, max_norm, eps, norm.data_ptr(), workspace.data_ptr())
    except RuntimeError:
        _explain_overlap(entries)  # (the library refuses it; sorting here would cost every call)
        raise
    _wrote(to if len(to) == count else [d for d in to if d is not None])
    return norm

"""Ids and the log-probabilities a network gives them: atom types - the 119 classes of ``atom_pred``, of which
model1.py:991-997 takes the types and generation.py:162-233 the softmax - or the tokens of any vocabulary.

* ``embed_tokens`` / ``embed_tokens_grad``: lookup of ids in a table with a scale, and the table's gradient;
* ``token_logprobs``: log-probabilities of chosen ids (scoring under a reference or an earlier policy);
* ``preference_loss``: pairs of molecules of which one is preferred;
* ``policy_loss``: rewards, with a clipped ratio to the policy that sampled and a KL term to a reference.

All run in the HIP library on the current stream of the tensors' device; there is no CPU path.  Logits and tables are
fp32, bf16 or fp16 with rows any distance apart; ids are int32 or int64.  An id outside the vocabulary (-1 by custom) is an
ignored position: a row of zeros, log-probability 0, no part in a loss.  The losses come in two forms: differentiable
(``loss.backward()``), and ``*_and_grad``, which returns the gradient of the logits beside the loss - a training step that
owns its backward pass hands it on with ``logits.backward(d_logits)`` and saves reading the logits again.  Second and
forward-mode derivatives are refused.
The reference has no counterpart (one-hot types, no loss on the distribution of ``atom_pred``)."""
import ctypes as C
from collections import namedtuple
from functools import lru_cache

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import PolicyArgs, PreferenceArgs, TokenArgs, check

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_TOKEN_BYTES = {torch.int32: 4, torch.int64: 8}
_INT_MAX = 0x7fffffff      # what the library's 32-bit sizes hold (a larger number would arrive as its low half)

PreferenceLoss = namedtuple("PreferenceLoss", "loss log_ratio margin")
PreferenceGrad = namedtuple("PreferenceGrad", "loss log_ratio margin d_logits")
PolicyLoss = namedtuple("PolicyLoss", "loss surrogate kl clip_fraction logp")
PolicyGrad = namedtuple("PolicyGrad", "loss surrogate kl clip_fraction logp d_logits")


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


class _on:
    """Makes a tensor's device the current one (free when it already is) and gives its current stream."""
    __slots__ = ("index", "back")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        now = torch.cuda.current_device()
        self.back = None
        if self.index != now:
            torch.cuda.set_device(self.index)
            self.back = now
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.back is not None:
            torch.cuda.set_device(self.back)


@lru_cache(maxsize=256)
def _workspace_bytes(entry, *sizes):
    return getattr(_lib.load(), entry)(*sizes)


def _check_tangent(t, name):
    """A tangent would be lost without a word: the kernels read the values only."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name} carries a tangent: forward-mode derivatives are not implemented")


def _check_float(t, name):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on a HIP device: the hot path has no CPU implementation")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be fp32, bf16 or fp16, got {t.dtype}")
    _check_tangent(t, name)


def _check_ids(tokens, device, name="tokens"):
    if tokens.dtype not in _TOKEN_BYTES:
        raise ValueError(f"{name} must be int32 or int64, got {tokens.dtype}")
    if tokens.device != device:
        raise ValueError(f"{name} lives on {tokens.device}, the other tensors on {device}")


def _rows(t, width):
    """[..., width] as rows with unit stride: (tensor to keep alive, number of rows, elements between rows)."""
    n = t.numel() // width
    if t.is_contiguous():
        return t, n, width
    if t.dim() != 2:
        t = t.reshape(n, width)
    if n <= 1 or width == 1 or t.stride(1) != 1 or t.stride(0) < width:   # transposed, or rows that overlap (expanded)
        return t.contiguous(), n, width
    return t, n, t.stride(0)


def _vector(t, n, device, name):
    """A [n] fp32 vector beside the logits (log-probabilities, advantages)."""
    if t.device != device:
        raise ValueError(f"{name} lives on {t.device}, the logits on {device}")
    if t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} elements, expected {n}")
    _check_tangent(t, name)
    if t.dtype != torch.float32:
        if t.dtype not in _DTYPES and t.dtype != torch.float64:
            raise ValueError(f"{name} must be a floating-point tensor, got {t.dtype}")
        t = t.float()
    return t.contiguous()


def _ptr_vector(seq_ptr, device, name="seq_ptr"):
    if seq_ptr.dtype not in _TOKEN_BYTES or seq_ptr.dim() != 1 or not 2 <= seq_ptr.numel() <= _INT_MAX:
        raise ValueError(f"{name} must be a 1-D int32 or int64 tensor of first positions, one more than there are sequences")
    if seq_ptr.device != device:
        raise ValueError(f"{name} lives on {seq_ptr.device}, the logits on {device}")
    if seq_ptr.dtype != torch.int32:   # (offsets beyond every position stay so)
        seq_ptr = seq_ptr.clamp(-_INT_MAX - 1, _INT_MAX).to(torch.int32)
    return seq_ptr.contiguous()


def _finite_scale(value, name):
    value = float(value)
    if not abs(value) <= 3e38:
        raise ValueError(f"{name} must be a finite number")
    return value


def _denominator(value):
    """0 (the count that the library takes itself) for None."""
    if value is None:
        return 0.0
    value = float(value)
    if not 2.0 ** -126 <= value <= 3e38:   # (what fp32 rounds to 0 would ask for the count)
        raise ValueError("denominator must be positive, and a normal number of fp32")
    return value


# ------------------------------------------------------------------------------------------------ embedding
def _embed(tokens, table, scale):
    _check_float(table, "table")
    if table.dim() != 2 or table.numel() == 0 or table.shape[1] > _INT_MAX:
        raise ValueError("table must be [rows, width], not empty and less than 2^31 wide")
    dev = table.device
    _check_ids(tokens, dev)
    scale = _finite_scale(scale, "scale")
    V, D = table.shape
    table, _, stride = _rows(table, D)
    ids = tokens.contiguous()
    out = torch.empty((*tokens.shape, D), dtype=table.dtype, device=dev)
    with _on(dev) as stream:
        check(_lib.load().ligdiff_embed(table.data_ptr(), _DTYPES[table.dtype], V, D, stride, ids.data_ptr(),
                                        _TOKEN_BYTES[ids.dtype], ids.numel(), scale, out.data_ptr(), D, stream), "ligdiff_embed")
    return out


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale):
        ctx.save_for_backward(tokens)
        ctx.rows, ctx.scale = table.shape[0], scale
        return _embed(tokens, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        return None, embed_tokens_grad(d_out, ctx.saved_tensors[0], ctx.rows, ctx.scale), None


def embed_tokens(tokens, table, scale=1.0):
    """``scale * table[tokens]`` [..., width] in the table's type; differentiable with respect to ``table``."""
    if torch.is_grad_enabled() and table.requires_grad:
        return _EmbedTokens.apply(tokens, table, scale)
    return _embed(tokens, table, scale)


def embed_tokens_grad(d_out, tokens, n_rows, scale=1.0, out=None, accumulate=False):
    """The gradient of ``embed_tokens`` with respect to the table: [n_rows, width], row v the scaled sum of the rows of
    ``d_out`` whose token is v.  ``out``: a tensor to write, of d_out's type or fp32 (``accumulate``: to add to, e.g. the
    fp32 gradient of a half-precision table over several micro-batches)."""
    _check_float(d_out, "d_out")
    dev = d_out.device
    _check_ids(tokens, dev)
    scale, n_rows = _finite_scale(scale, "scale"), int(n_rows)
    D = d_out.shape[-1] if d_out.dim() else 0
    if n_rows < 1 or not 1 <= D <= _INT_MAX or d_out.shape[:-1] != tokens.shape:
        raise ValueError("d_out must be [*tokens.shape, width] with width (below 2^31) and n_rows at least 1")
    rows, n, stride = _rows(d_out, D)
    ids = tokens.contiguous()
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs the tensor to add to (out)")
        out = torch.empty((n_rows, D), dtype=d_out.dtype, device=dev)
    elif out.shape != (n_rows, D) or out.device != dev or out.dtype not in (d_out.dtype, torch.float32):
        raise ValueError(f"out must be [{n_rows}, {D}] on {dev}, of d_out's type or fp32")
    elif (D > 1 and out.stride(1) != 1) or (n_rows > 1 and out.stride(0) < D):
        raise ValueError("out must have rows of unit stride that do not overlap")
    else:
        _check_tangent(out, "out")
    lib = _lib.load()
    nbytes = _workspace_bytes("ligdiff_embed_grad_workspace_bytes", n, n_rows, D)
    with _on(dev) as stream:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        check(lib.ligdiff_embed_grad(rows.data_ptr(), _DTYPES[rows.dtype], stride, ids.data_ptr(), _TOKEN_BYTES[ids.dtype], n,
                                     n_rows, D, scale, out.data_ptr(), _DTYPES[out.dtype], out.stride(0) if n_rows > 1 else D,
                                     1 if accumulate else 0, ws.data_ptr(), nbytes, stream), "ligdiff_embed_grad")
    return out


# ------------------------------------------------------------------------------------------------ log-probabilities
def _check_rows(logits, tokens, temperature):
    _check_float(logits, "logits")
    if logits.dim() < 2 or not 1 <= logits.shape[-1] <= _INT_MAX:
        raise ValueError("logits must be [..., vocabulary] with fewer than 2^31 ids")
    _check_ids(tokens, logits.device)
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} do not match logits {tuple(logits.shape)}")
    if not 1e-20 <= float(temperature) <= 1e20:
        raise ValueError("temperature must be between 1e-20 and 1e20")


def _token_args(logits, tokens, temperature):
    """(struct, rows, ids, n, V) of checked tensors, which must outlive the call."""
    V = logits.shape[-1]
    rows, n, stride = _rows(logits, V)
    ids = tokens.contiguous()
    return TokenArgs(rows.data_ptr(), ids.data_ptr(), stride, n, V, _DTYPES[rows.dtype], _TOKEN_BYTES[ids.dtype],
                     float(temperature)), rows, ids, n, V


def _logprob(logits, tokens, temperature, want_stats):
    _check_rows(logits, tokens, temperature)
    a, rows, ids, n, V = _token_args(logits, tokens, temperature)
    dev = logits.device
    logp = torch.empty(tokens.shape, dtype=torch.float32, device=dev)
    stats = torch.empty(n, 2, dtype=torch.float32, device=dev) if want_stats else None
    with _on(dev) as stream:
        check(_lib.load().ligdiff_token_logprob(C.byref(a), logp.data_ptr(), stats.data_ptr() if want_stats else None, stream),
              "ligdiff_token_logprob")
    return logp, stats


def _logprob_grad(logits, tokens, temperature, stats, coef, index=None, upstream=None):
    a, rows, ids, n, V = _token_args(logits, tokens, temperature)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    with _on(logits.device) as stream:
        check(_lib.load().ligdiff_token_logprob_grad(C.byref(a), stats.data_ptr(), coef.data_ptr(),
                                                     None if index is None else index.data_ptr(), coef.numel(), 1.0,
                                                     None if upstream is None else upstream.data_ptr(), d.data_ptr(), V, stream),
              "ligdiff_token_logprob_grad")
    return d


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature):
        logp, stats = _logprob(logits, tokens, temperature, True)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.temperature = temperature
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, tokens, stats = ctx.saved_tensors
        return _logprob_grad(logits, tokens, ctx.temperature, stats, g.float().contiguous()), None, None


def token_logprobs(logits, tokens, temperature=1.0):
    """fp32 log softmax(logits / temperature) at ``tokens`` (the leading shape of ``logits``), 0 at ignored positions;
    differentiable with respect to ``logits``."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLogprobs.apply(logits, tokens, temperature)
    return _logprob(logits, tokens, temperature, False)[0]


# ------------------------------------------------------------------------------------------------ preference loss
def _preference_inputs(logits, tokens, seq_ptr, ref_logp, beta, label_smoothing, kind, temperature, denominator, grad_scale):
    """Checks what a preference loss is given, of the logits only where they are and their type and shape:
    (seq_ptr, ref_logp, denominator, grad_scale) as the library takes them."""
    if kind not in _lib.PREFERENCE_KINDS:
        raise ValueError(f"kind must be one of {sorted(_lib.PREFERENCE_KINDS)}")
    beta, label_smoothing = float(beta), float(label_smoothing)
    if not 0.0 < beta <= 3e38 or not 0.0 <= label_smoothing < 0.5:
        raise ValueError("beta must be positive and label_smoothing in [0, 0.5)")
    if kind != "sigmoid" and label_smoothing:
        raise ValueError("label_smoothing belongs to the sigmoid loss")
    _check_rows(logits, tokens, temperature)
    dev = logits.device
    ptr = _ptr_vector(seq_ptr, dev)
    if ptr.numel() % 2 != 1:
        raise ValueError("seq_ptr must hold an even number of sequences: the preferred ones, then the others in the same order")
    ref = None if ref_logp is None else _vector(ref_logp, tokens.numel(), dev, "ref_logp")
    return ptr, ref, _denominator(denominator), _finite_scale(grad_scale, "grad_scale")


def _preference(logits, tokens, seq_ptr, ref_logp, beta, label_smoothing, kind, average, temperature, denominator, grad_scale,
                want_grad):
    ptr, ref, denominator, grad_scale = _preference_inputs(logits, tokens, seq_ptr, ref_logp, beta, label_smoothing, kind,
                                                           temperature, denominator, grad_scale)
    a, rows, ids, n, V = _token_args(logits, tokens, temperature)
    dev, P = logits.device, (ptr.numel() - 1) // 2
    lib = _lib.load()
    nbytes = _workspace_bytes("ligdiff_preference_workspace_bytes", n, P)
    f32 = dict(dtype=torch.float32, device=dev)
    with _on(dev) as stream:
        loss, log_ratio, margin = torch.empty((), **f32), torch.empty(2 * P, **f32), torch.empty(P, **f32)
        slope = stats = row_seq = d = None
        if want_grad:   # what only a later gradient needs lies behind the workspace
            d = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
            ws = torch.empty(nbytes + 8 * P + 12 * n, dtype=torch.uint8, device=dev)
            at = ws.data_ptr() + nbytes
            saved = (at, at + 8 * P, at + 8 * P + 8 * n)
        else:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            slope, stats, row_seq = torch.empty(2 * P, **f32), torch.empty(n, 2, **f32), torch.empty(n, dtype=torch.int32, device=dev)
            saved = (slope.data_ptr(), stats.data_ptr(), row_seq.data_ptr())
        q = PreferenceArgs(ptr.data_ptr(), None if ref is None else ref.data_ptr(), P, _lib.PREFERENCE_KINDS[kind],
                           1 if average else 0, float(beta), float(label_smoothing), denominator, grad_scale, loss.data_ptr(),
                           log_ratio.data_ptr(), margin.data_ptr(), *saved,
                           None if d is None else d.data_ptr(), V, ws.data_ptr(), nbytes)
        check(lib.ligdiff_preference_loss(C.byref(a), C.byref(q), stream), "ligdiff_preference_loss")
    return loss, log_ratio, margin, slope, stats, row_seq, d


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, seq_ptr, ref_logp, opts):
        loss, log_ratio, margin, slope, stats, row_seq, _ = _preference(logits, tokens, seq_ptr, ref_logp, *opts, 1.0, False)
        ctx.save_for_backward(logits, tokens, slope, stats, row_seq)
        ctx.temperature = opts[4]
        ctx.mark_non_differentiable(log_ratio, margin)
        return loss, log_ratio, margin

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        logits, tokens, slope, stats, row_seq = ctx.saved_tensors
        return _logprob_grad(logits, tokens, ctx.temperature, stats, slope, row_seq, g.float().contiguous()), None, None, None, None


def preference_loss(logits, tokens, seq_ptr, ref_logp=None, beta=0.1, label_smoothing=0.0, kind="sigmoid", average=False,
                    temperature=1.0, denominator=None):
    """Preference loss over pairs of sequences: of the 2 P sequences that ``seq_ptr`` [2 P + 1] delimits (``mol_ptr`` of a
    packed batch), number p is preferred over number P + p.  With r the sum over a sequence of logp - ref_logp (its mean
    with ``average``) and d = r_p - r_{P+p}:

        kind "sigmoid": -(1 - e) log sigmoid(beta d) - e log sigmoid(-beta d), e = label_smoothing
        kind "ipo":     (d - 1 / (2 beta))^2

    averaged over the pairs, or summed and divided by ``denominator`` (data parallel: the pairs of all ranks).
    Returns (loss, log_ratio [2 P], margin [P]); ``loss`` is differentiable with respect to ``logits``."""
    opts = (beta, label_smoothing, kind, average, temperature, denominator)
    if torch.is_grad_enabled() and logits.requires_grad:
        return PreferenceLoss(*_PreferenceLoss.apply(logits, tokens, seq_ptr, ref_logp, opts))
    return PreferenceLoss(*_preference(logits, tokens, seq_ptr, ref_logp, *opts, 1.0, False)[:3])


def preference_loss_and_grad(logits, tokens, seq_ptr, ref_logp=None, beta=0.1, label_smoothing=0.0, kind="sigmoid",
                             average=False, temperature=1.0, denominator=None, grad_scale=1.0):
    """``preference_loss`` and ``d_logits`` = grad_scale * d loss / d logits, in the logits' type."""
    loss, log_ratio, margin, _, _, _, d = _preference(logits, tokens, seq_ptr, ref_logp, beta, label_smoothing, kind, average,
                                                      temperature, denominator, grad_scale, True)
    return PreferenceGrad(loss, log_ratio, margin, d)


# ------------------------------------------------------------------------------------------------ policy loss
def _policy_inputs(logits, tokens, seq_ptr, advantage, old_logp, ref_logp, advantage_per, clip_low, clip_high, kl_coef, aggregate,
                   temperature, denominator, grad_scale):
    """Checks what a policy loss is given, of the logits only where they are and their type and shape:
    (seq_ptr, number of sequences, advantage, old_logp, ref_logp, denominator, grad_scale) as the library takes them."""
    if aggregate not in _lib.POLICY_MEANS:
        raise ValueError(f"aggregate must be one of {sorted(_lib.POLICY_MEANS)}")
    clip_low, clip_high, kl_coef = float(clip_low), float(clip_high), float(kl_coef)
    if not 0.0 <= clip_low <= 1.0 or not 0.0 <= clip_high <= 3e38 or not 0.0 <= kl_coef <= 3e38:
        raise ValueError("clip_low must be in [0, 1], clip_high and kl_coef at least 0")
    _check_rows(logits, tokens, temperature)
    dev, n = logits.device, tokens.numel()
    ptr = None if seq_ptr is None else _ptr_vector(seq_ptr, dev)
    S = 1 if ptr is None else ptr.numel() - 1
    if advantage_per not in ("sequence", "token"):
        raise ValueError("advantage_per must be 'sequence' or 'token'")
    adv = _vector(advantage, n if advantage_per == "token" else S, dev, "advantage")
    old = None if old_logp is None else _vector(old_logp, n, dev, "old_logp")
    ref = None if ref_logp is None else _vector(ref_logp, n, dev, "ref_logp")
    return ptr, S, adv, old, ref, _denominator(denominator), _finite_scale(grad_scale, "grad_scale")


def _policy(logits, tokens, seq_ptr, advantage, old_logp, ref_logp, advantage_per, clip_low, clip_high, kl_coef, aggregate,
            temperature, denominator, grad_scale, want_grad, want_saved):
    ptr, S, adv, old, ref, denominator, grad_scale = _policy_inputs(logits, tokens, seq_ptr, advantage, old_logp, ref_logp,
                                                                    advantage_per, clip_low, clip_high, kl_coef, aggregate,
                                                                    temperature, denominator, grad_scale)
    a, rows, ids, n, V = _token_args(logits, tokens, temperature)
    dev = logits.device
    mean = _lib.POLICY_MEANS[aggregate]
    lib = _lib.load()
    nbytes = _workspace_bytes("ligdiff_policy_workspace_bytes", n, S, mean)
    f32 = dict(dtype=torch.float32, device=dev)
    with _on(dev) as stream:
        result, logp = torch.empty(4, **f32), torch.empty(tokens.shape, **f32)
        stats, coef = (torch.empty(n, 2, **f32), torch.empty(n, **f32)) if want_saved else (None, None)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        d = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if want_grad else None
        q = PolicyArgs(None if ptr is None else ptr.data_ptr(), adv.data_ptr(), None if old is None else old.data_ptr(),
                       None if ref is None else ref.data_ptr(), S, 1 if advantage_per == "token" else 0, mean, float(clip_low), float(clip_high),
                       float(kl_coef), denominator, grad_scale, result.data_ptr(), logp.data_ptr(), stats.data_ptr() if want_saved else None,
                       coef.data_ptr() if want_saved else None, None if d is None else d.data_ptr(), V, ws.data_ptr(), nbytes)
        check(lib.ligdiff_policy_loss(C.byref(a), C.byref(q), stream), "ligdiff_policy_loss")
    return result, logp, stats, coef, d


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, seq_ptr, advantage, old_logp, ref_logp, opts):
        result, logp, stats, coef, _ = _policy(logits, tokens, seq_ptr, advantage, old_logp, ref_logp, *opts, 1.0, False, True)
        ctx.save_for_backward(logits, tokens, stats, coef)
        ctx.temperature = opts[5]
        loss, rest = result[0].clone(), result[1:]
        ctx.mark_non_differentiable(rest, logp)
        return loss, rest, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *_):
        logits, tokens, stats, coef = ctx.saved_tensors
        return (_logprob_grad(logits, tokens, ctx.temperature, stats, coef, None, g.float().contiguous()),) + (None,) * 6


def policy_loss(logits, tokens, seq_ptr, advantage, old_logp=None, ref_logp=None, advantage_per="sequence", clip_low=0.2,
                clip_high=0.2, kl_coef=0.0, aggregate="token", temperature=1.0, denominator=None):
    """Clipped policy loss with a KL term.  With rho = exp(logp - old_logp) (1 without ``old_logp``) and
    k = ref_logp - logp, a position contributes

        -min(rho A, clip(rho, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(k) - k - 1)

    ``advantage``: A, one value for each sequence, or for each position with ``advantage_per`` "token".
    ``seq_ptr`` [S + 1] delimits the sequences (None: one); positions outside take no part.  ``aggregate`` "token": mean
    over the positions that take part; "sequence": mean over the sequences of each one's mean.  ``denominator`` takes the
    place of the number of positions / sequences (data parallel).  Returns (loss, surrogate, kl, clip_fraction, logp);
    ``loss`` is differentiable with respect to ``logits``."""
    opts = (advantage_per, clip_low, clip_high, kl_coef, aggregate, temperature, denominator)
    if torch.is_grad_enabled() and logits.requires_grad:
        loss, rest, logp = _PolicyLoss.apply(logits, tokens, seq_ptr, advantage, old_logp, ref_logp, opts)
        return PolicyLoss(loss, *rest.unbind(0), logp)
    result, logp, _, _, _ = _policy(logits, tokens, seq_ptr, advantage, old_logp, ref_logp, *opts, 1.0, False, False)
    return PolicyLoss(*result.unbind(0), logp)


def policy_loss_and_grad(logits, tokens, seq_ptr, advantage, old_logp=None, ref_logp=None, advantage_per="sequence",
                         clip_low=0.2, clip_high=0.2, kl_coef=0.0, aggregate="token", temperature=1.0, denominator=None,
                         grad_scale=1.0):
    """``policy_loss`` and ``d_logits`` = grad_scale * d loss / d logits, from one pass over the logits."""
    result, logp, _, _, d = _policy(logits, tokens, seq_ptr, advantage, old_logp, ref_logp, advantage_per, clip_low, clip_high,
                                    kl_coef, aggregate, temperature, denominator, grad_scale, True, False)
    return PolicyGrad(*result.unbind(0), logp, d)

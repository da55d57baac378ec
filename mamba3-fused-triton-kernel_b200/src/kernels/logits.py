"""What a decode step does with its logits (``m3_process_logits``,
``m3_next_tokens``).

``process_logits`` adjusts a (B, V) matrix of logits by a row's history of
tokens, a bias and a mask of allowed tokens; ``next_tokens`` makes the same
adjustments and returns the next token of every row with its log-probability,
without storing the adjusted logits.  In fp32, in this order:

    token in tokens[b, :length]        z = z / repetition if z > 0 else z * repetition
    c times in tokens[b, prompt:length]    z = z - frequency * c
    c > 0                              z = z - presence
    always                             z = z + bias
    not allowed                        z = -inf

The reference's decode ends at the layer output; none of this has a
counterpart there.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from src import _native as nat

_CODE = {torch.float32: nat.M3_F32, torch.bfloat16: nat.M3_BF16}
_INTS = {torch.int32: 0, torch.int64: 1}

PerRow = Union[float, torch.Tensor, None]

_host_process = _host_next = None  # the host module's functions, once looked up


def _per_row(name: str, value: PerRow, neutral: float, B: int, dev: int, keep: list) -> tuple:
    """(pointer, scalar) of a per-row fp32 value: a (B,) tensor, or a number
    for all rows."""
    if not isinstance(value, torch.Tensor):
        return 0, float(value)
    assert value.shape == (B,) and value.get_device() == dev and value.is_floating_point(), \
        f"{name} must be a number or a float ({B},) tensor on the logits' device"
    if value.dtype != torch.float32 or not value.is_contiguous():
        value = value.float().contiguous()
        keep.append(value)
    return value.data_ptr(), neutral


def _row_ints(name: str, value: torch.Tensor, B: int, dev: int, keep: list) -> tuple:
    """(pointer, is int64) of a (B,) integer tensor."""
    i64 = _INTS.get(value.dtype)
    assert i64 is not None and value.shape == (B,) and value.get_device() == dev, \
        f"{name} must be an int32 or int64 ({B},) tensor on the logits' device"
    if not value.is_contiguous():
        value = value.contiguous()
        keep.append(value)
    return value.data_ptr(), i64


def _shared_rows(name: str, value: torch.Tensor, dtype: torch.dtype, B: int, width: int, dev: int,
                 keep: list) -> tuple:
    """(pointer, row stride) of a (width,) or (B, width) tensor."""
    shape = value.shape
    assert value.get_device() == dev and len(shape) in (1, 2) and shape[-1] >= width and \
        (len(shape) == 1 or shape[0] == B or shape[0] == 1), \
        f"{name} must be ({width},) or ({B}, {width}) on the logits' device, got {tuple(shape)}"
    if value.dtype != dtype or (value.stride(-1) != 1 and width > 1):
        value = value.to(dtype).contiguous()
        keep.append(value)
    return value.data_ptr(), value.stride(0) if len(shape) == 2 and shape[0] > 1 else 0


def _refuse_gradients(*values) -> None:
    if nat.wants_gradient(*(v for v in values if isinstance(v, torch.Tensor))):
        raise RuntimeError("the logit operators have no gradient: call them under torch.no_grad() or detach")


def _adjust_args(logits, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty, frequency_penalty,
                 bias, allowed, keep: list) -> tuple:
    """Checked arguments that both entry points share: the packed fields up
    to ``allowed``, with the sampling ones open."""
    dev = logits.get_device() if logits.is_cuda else -1
    assert dev >= 0 and logits.dim() == 2, "logits must be a (B, V) CUDA tensor"
    B, V = logits.shape
    code = _CODE.get(logits.dtype)
    assert code is not None, f"logits must be float32 or bfloat16 (got {logits.dtype})"
    _refuse_gradients(logits, bias, repetition_penalty, presence_penalty, frequency_penalty)
    if logits.is_contiguous():
        ld = V
    else:
        if logits.stride(1) != 1 and V > 1:
            logits = logits.contiguous()
            keep.append(logits)
        ld = logits.stride(0)
    T = t_ptr = t_stride = t_i64 = len_ptr = len_i64 = pro_ptr = pro_i64 = 0
    if tokens is not None:
        t_i64 = _INTS.get(tokens.dtype)
        shape = tokens.shape
        assert t_i64 is not None and len(shape) == 2 and shape[0] == B and tokens.get_device() == dev, \
            f"tokens must be an int32 or int64 ({B}, T) tensor on the logits' device"
        T = shape[1]
        if tokens.is_contiguous():
            t_stride = T
        else:
            if tokens.stride(1) != 1 and T > 1:
                tokens = tokens.contiguous()
                keep.append(tokens)
            t_stride = tokens.stride(0)
        t_ptr = tokens.data_ptr()
        if lengths is not None:
            len_ptr, len_i64 = _row_ints("lengths", lengths, B, dev, keep)
        if prompt_lengths is not None:
            pro_ptr, pro_i64 = _row_ints("prompt_lengths", prompt_lengths, B, dev, keep)
    else:
        assert lengths is None and prompt_lengths is None, "lengths and prompt_lengths go with tokens"
    rep = pres = freq = mask_ptr = mask_stride = bias_ptr = bias_stride = 0
    rep_value, pres_value, freq_value = 1.0, 0.0, 0.0
    if repetition_penalty is not None:
        rep, rep_value = _per_row("repetition_penalty", repetition_penalty, 1.0, B, dev, keep)
        if not rep_value > 0:
            raise ValueError(f"repetition_penalty must be above 0 (got {rep_value})")
    if presence_penalty is not None:
        pres, pres_value = _per_row("presence_penalty", presence_penalty, 0.0, B, dev, keep)
    if frequency_penalty is not None:
        freq, freq_value = _per_row("frequency_penalty", frequency_penalty, 0.0, B, dev, keep)
    if bias is not None:
        assert bias.is_floating_point(), "bias must be a float tensor"
        bias_ptr, bias_stride = _shared_rows("bias", bias, torch.float32, B, V, dev, keep)
    if allowed is not None:
        assert allowed.dtype == torch.int32, "allowed must hold the mask's bits in int32 words"
        mask_ptr, mask_stride = _shared_rows("allowed", allowed, torch.int32, B, -(-V // 32), dev, keep)
    return (dev, B, V,
            (B, V, T, code, logits.data_ptr(), ld, t_ptr, t_stride, len_ptr, pro_ptr, t_i64, len_i64, pro_i64),
            (rep, pres, freq, rep_value, pres_value, freq_value), (bias_ptr, bias_stride, mask_ptr, mask_stride))


def process_logits(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None, prompt_lengths: Optional[torch.Tensor] = None, *,
                   repetition_penalty: PerRow = None, presence_penalty: PerRow = None,
                   frequency_penalty: PerRow = None, bias: Optional[torch.Tensor] = None,
                   allowed: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Adjusted logits, computed in fp32 and rounded once.

    logits  (B, V) float32 or bfloat16, any row stride
    tokens  (B, T) int32 or int64, the rows' histories; ids outside [0, V)
            (padding) are skipped
    lengths (B,) entries of each history in use (clamped to T; all without it)
    prompt_lengths (B,) of those, how many came from the prompt: they count
            as seen, not as generated (0 without it)
    repetition_penalty, presence_penalty, frequency_penalty
            a number, or a float (B,) tensor
    bias    (V,) or (B, V), read as float32
    allowed (W,) or (B, W) int32, W at least ceil(V / 32): bit i % 32 of word
            i // 32 says whether token i may follow
    out     (B, V) float32 or bfloat16, unit column stride; ``logits`` itself
            works in place.  It overlaps no other argument.  A new tensor of
            the logits' type without it.

    Penalties given as tensors are not looked at by the host: a repetition
    penalty is above 0.  Inference only: logits, a bias, penalties or an out
    that ask for a gradient, also a forward-mode one, are refused."""
    global _host_process
    if out is None:
        if _host_process is None:
            _host_process = nat.host_entry("process_logits")
        y = _host_process(logits, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty,
                          frequency_penalty, bias, allowed)
        if y is not None:
            return y
    keep: list = []
    dev, B, V, head, mid, tail = _adjust_args(logits, tokens, lengths, prompt_lengths, repetition_penalty,
                                              presence_penalty, frequency_penalty, bias, allowed, keep)
    out_ld = V
    if out is None:
        out = torch.empty((B, V), dtype=logits.dtype, device=logits.device)
    else:
        assert out.shape == logits.shape and out.device == logits.device and out.dtype in _CODE, \
            f"out must be a float32 or bfloat16 {(B, V)} tensor on the logits' device"
        assert (V <= 1 or out.stride(1) == 1) and (B <= 1 or out.stride(0) >= V), \
            "out must have unit column stride and rows that do not overlap"
        _refuse_gradients(out)
        if out is not logits and _overlap(out, logits):
            assert out.data_ptr() == logits.data_ptr() and out.dtype == logits.dtype and \
                out.stride() == logits.stride(), "out may be the logits themselves, not overlap them otherwise"
        if B > 1:
            out_ld = out.stride(0)
    if B == 0 or V == 0:
        return out
    nat.call("m3_process_logits", nat.LOGITS_ARGS.pack(
        *head, 0, *mid, 0.0, *tail, out.data_ptr(), out_ld, _CODE[out.dtype], 0, 0, 0, 0, 0, 0),
        dev)
    return out


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two (B, V) tensors may share memory.  Rows at the same
    distance are told apart (parts of the columns of one buffer); others go
    by their first and last bytes."""
    def span(t):
        if t.numel() == 0:
            return 0, 0
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    if not (a0 < b1 and b0 < a1):
        return False
    pitch = a.stride(0) * a.element_size()
    if a.shape[0] == 1 or pitch == 0 or pitch != b.stride(0) * b.element_size() or \
            (a.shape[1] > 1 and (a.stride(1) != 1 or b.stride(1) != 1)):
        return True
    at = (b0 - a0) % pitch  # b's rows from a's
    return at < a.shape[1] * a.element_size() or at + b.shape[1] * b.element_size() > pitch


def next_tokens(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None, prompt_lengths: Optional[torch.Tensor] = None, *,
                repetition_penalty: PerRow = None, presence_penalty: PerRow = None,
                frequency_penalty: PerRow = None, bias: Optional[torch.Tensor] = None,
                allowed: Optional[torch.Tensor] = None, temperature: PerRow = None,
                seeds: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None) -> tuple:
    """(ids (B,) int64, logprobs (B,) float32): every row's next token.

    The arguments of ``process_logits``, and

    temperature  None: greedy, the largest adjusted logit, the lowest index
                 among equals.  A number or a float (B,) tensor: rows with a
                 temperature above 0 are drawn from softmax(z / temperature),
                 the others are greedy.
    seeds        (B,) int64, with a temperature: the row's random stream
    positions    (B,) int64, the place in it (0 without it): a row's draw
                 depends on its logits, seed and position only, so a position
                 that advances with the row's length gives a new draw a step

    ``logprobs`` is the token's log-probability under the distribution the
    row was drawn from (greedy rows: at temperature 1).  A NaN that is not
    masked is taken as the largest, with logprob NaN; a row with nothing
    allowed gives token 0 with logprob -inf."""
    global _host_next
    if _host_next is None:
        _host_next = nat.host_entry("next_tokens")
    both = _host_next(logits, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty,
                      frequency_penalty, bias, allowed, temperature, seeds, positions)
    if both is not None:
        return both
    keep: list = []
    dev, B, V, head, mid, tail = _adjust_args(logits, tokens, lengths, prompt_lengths, repetition_penalty,
                                              presence_penalty, frequency_penalty, bias, allowed, keep)
    assert V > 0, "next_tokens needs at least one logit a row"
    sample = 0
    temp, temp_value = 0, 0.0
    seed_ptr = pos_ptr = 0
    if temperature is not None:
        sample = 1
        _refuse_gradients(temperature)
        temp, temp_value = _per_row("temperature", temperature, 0.0, B, dev, keep)
        assert seeds is not None, "a temperature needs seeds"
        assert seeds.dtype == torch.int64 and (positions is None or positions.dtype == torch.int64), \
            "seeds and positions must be int64"
        seed_ptr, _ = _row_ints("seeds", seeds, B, dev, keep)
        if positions is not None:
            pos_ptr, _ = _row_ints("positions", positions, B, dev, keep)
    device = logits.device
    ids = torch.empty((B,), dtype=torch.int64, device=device)
    logprobs = torch.empty((B,), dtype=torch.float32, device=device)
    if B > 0:
        nat.call("m3_next_tokens", nat.LOGITS_ARGS.pack(
            *head, sample, *mid, temp_value, *tail, 0, 0, 0, 0, temp, seed_ptr, pos_ptr, ids.data_ptr(),
            logprobs.data_ptr()), dev)
    return ids, logprobs

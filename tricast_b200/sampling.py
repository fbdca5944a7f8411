"""The next tokens from their logits and given random numbers. No TriCast counterpart."""

from __future__ import annotations

import torch

from . import _native as N


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature=1.0, top_k=None, top_p=None, min_p=None,
                  return_logprobs: bool = False):
    """One token (int64) for each row of ``logits`` ``[rows, vocab]`` (any row stride), chosen by ``uniform`` (fp32 ``[rows]`` in
    ``[0, 1)``).

    Settings are numbers (taken as fp32), or tensors with one a row (fp32; ``top_k`` int32); ``None`` leaves a filter out. A token weighs
    ``w = exp((l - max l) / temperature)``, 0 where that is below ``2**-126``. Of the tokens with a weight the ``top_k`` largest logits
    stay (ties: the lower index; 0 or less: all), of those, in descending order, the fewest whose weights reach ``top_p`` of
    their sum (1 or more: all), of those the ones with ``w >= min_p`` (the largest always stays). The token is the first index
    at which the sum of what stayed, in index order, exceeds ``uniform`` times the total. ``temperature`` 0 or less takes
    the first largest logit. Temperatures between 0 and ``2**-100`` count as that.

    A row that has no logit above ``-inf`` gives ``-1`` (log-probability ``-inf``), one with a NaN ``-1`` (NaN). Settings that
    are NaN bound nothing (a temperature: 0). With ``return_logprobs`` also the fp32 logarithms of the tokens' shares of what
    stayed. Weights are fp32, within 1.3e-7 of themselves (without ``top_k`` and ``top_p`` fp64, 2e-10), and their sums fp64 in a
    fixed order: the same call gives the same tokens, and they are the definition's unless ``uniform`` or ``top_p`` lies within 1e-7 of a
    border of the shares, or a weight within 1.3e-7 of ``min_p``. No gradients pass."""
    if not logits.is_cuda:
        raise ValueError("the B200 backend requires a CUDA tensor")
    if logits.ndim != 2 or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, vocab] with a vocabulary that is not empty (at most 2**23)")
    rows, vocab = logits.shape
    device = logits.device
    dtype = N.dtype_code(logits.dtype)

    def setting(value, neutral, kind, name):
        """A pointer or None, and the number for every row."""
        if value is None:
            return None, neutral, None
        if not isinstance(value, torch.Tensor):
            return None, value, None
        if value.shape != (rows,) or value.dtype != kind or value.device != device:
            raise ValueError(f"{name} must be a number or a {str(kind)[6:]} tensor [rows] on the logits' device")
        value = value if value.stride(0) == 1 else value.contiguous()
        return value.data_ptr(), neutral, value

    u, _, u_kept = setting(uniform, 0.0, torch.float32, "uniform")
    if u_kept is None:
        raise ValueError("uniform must be a float32 tensor [rows] on the logits' device")
    t, t_all, t_kept = setting(temperature, 1.0, torch.float32, "temperature")
    k, k_all, k_kept = setting(top_k, 0, torch.int32, "top_k")
    p, p_all, p_kept = setting(top_p, 1.0, torch.float32, "top_p")
    m, m_all, m_kept = setting(min_p, 0.0, torch.float32, "min_p")
    k_all = max(0, min(int(k_all), vocab))
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    if rows > 1 and logits.stride(0) < vocab:
        logits = logits.contiguous()
    tokens = torch.empty(rows, dtype=torch.int64, device=device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=device) if return_logprobs else None
    index = device.index
    with N.on_device(index):
        status = N.lib().tc_sample_tokens(logits.data_ptr(), dtype, rows, vocab, logits.stride(0), u, t, t_all, k, k_all, p, p_all,
                                          m, m_all, tokens.data_ptr(), None if logprobs is None else logprobs.data_ptr(),
                                          N.raw_stream(index))
    if status:
        N.check(status, "tc_sample_tokens")
    return (tokens, logprobs) if return_logprobs else tokens


__all__ = ["sample_tokens"]

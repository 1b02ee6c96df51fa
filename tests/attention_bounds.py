"""How far the output of an attention may lie from its 64-bit definition when
its softmax weights keep the accuracy of FP32: the rounding of the result to
BF16 and what FP32 arithmetic leaves, nothing for the weights' own storage."""
import torch


def output_bound(out, spread, size, keys, d):
    """Of each output.  spread: sum of w |v|; size: per row, the largest sum of
    |q k| / sqrt(d) over the keys.

    A weight is off by its score's d FP32 accumulations (d 2^-24 of size, twice:
    in its numerator and in the denominator), by two BF16 numbers that are cut
    off (2^-14) and by exponential and quotient (2^-20); the second product
    accumulates `keys` terms (2^-23 each, which covers an accumulator that
    truncates).  All of it counts against spread.  The result is rounded to the
    nearest of BF16's 8-bit significands once."""
    delta = (2 * d * 2.0 ** -24 * size[..., None] + 2.0 ** -14 + 2.0 ** -20 + keys * 2.0 ** -23) * spread
    most = (out.abs() + delta).clamp(min=2.0 ** -126)
    return torch.exp2(torch.floor(torch.log2(most)) - 8) + delta

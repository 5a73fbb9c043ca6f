"""Two-key and many-key rows whose output is one weight, or the sum of many small ones:
what P's rounding to 16-bit parts leaves of it.  Nothing here needs a GPU.

P = 2^(x + 8) of a key whose score is x log2 units (x <= 0) below the row's largest, so
the largest weight has P = 256.  A part of P is the 16-bit value nearest to what the
parts before it leave."""
import torch

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def parts_of(cache_dtype, out):
    """(type, number) of the parts of P, as include/ncz_paged.h says."""
    if cache_dtype == E4M3:
        return F16, 1 if out == BF16 else 2
    return cache_dtype, 3 if cache_dtype == BF16 and out == F32 else 2


def in_parts(p, dtype, count):
    """What `count` parts of the float64 tensor p (rounded to f32) add up to."""
    left = p.float()
    total = torch.zeros_like(p)
    for _ in range(count):
        part = left.to(dtype).float()
        total += part.double()
        left = left - part
    return total


def weight_error(dtype, count):
    """(relative, absolute) bound of a weight in parts, the absolute one against the row's
    largest weight: half a step for each part, and for f16 its smallest step, 2^-24: a part is
    off by 2^-25 at least, where the largest P is 256 or more."""
    return (torch.finfo(dtype).eps / 2) ** count, 2.0 ** -33 if dtype == F16 else 0.0


# Rows of two keys: the first at a score of 0, with V = 0; the second at b, with V = 1, so
# that o = w / (1 + w), w = exp(b): the relative error of o is that of one weight.
def two_keys(cache_dtype):
    """Scores b in (-2, 0) of the second keys, values of the cache's type."""
    if cache_dtype == E4M3:
        bits = torch.arange(128, dtype=torch.int32).to(torch.uint8).view(E4M3).float()
        return -bits[(bits > 2.0 ** -4) & (bits < 2)]
    g = torch.Generator().manual_seed(7)
    return (-2 * torch.rand(400, generator=g) * 0.99 - 0.001).to(cache_dtype).float()


# Relative bound of such an o in f32 besides that of the weight: the exponent 8 + b log2 e, in
# [5, 8), is rounded once (2^-22) and log2 e by 2^-24 of up to 2.9 (2^-22.4), together 1.8 2^-22
# ln 2 = 1.25 2^-22; ex2 2^-22; up to three products into one sum, cut off at 2^-23 each, 1.5 2^-22;
# the sum 1 + w, the division and the last product 2^-23 each at most, 1.5 2^-22.  5.25 2^-22 in all.
TWO_KEYS_BOUND = 5.25 * 2.0 ** -22


# Rows of n keys: one at a score of 0 with V = 0, all others `down` log2 units below it with V = 1:
# o = (n - 1) w / (1 + (n - 1) w), w = 2^-down, a sum of n - 1 equal small weights.
def tail_want(n, score):
    """o in float64 for the score (natural log units) of the other keys."""
    w = torch.exp(torch.tensor(score, dtype=torch.float64))
    return float((n - 1) * w / (1 + (n - 1) * w)), float(w)


def tail_bound(n, w, want, dtype, count):
    """Each of the n - 1 weights is off by weight_error, and by 2^-17 of it: the exponents 8 and
    8 - down come from an offset below 64 in size that is rounded (2^-19), log2 e times the scale
    by 2^-24 of 40 and the product by 2^-19, ex2 by 2^-22: 2^-17.4 with the largest key's own.
    The sums are chains of at most n / 8 additions, 2^-23 each."""
    relative, absolute = weight_error(dtype, count)
    # a weight is one value: in f16 it is off by whichever of the two is larger
    each = max(relative * w, absolute)
    return (n - 1) * each + want * (2.0 ** -17 + n / 8 * 2.0 ** -23)

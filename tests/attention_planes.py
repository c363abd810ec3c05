"""Inputs of attention in float32 whose results show every bit of the products (not collected by pytest).

The kernels take a float x as x0 + x1 + x2, each the rounding to 16 bits (bfloat16) of what those before it leave: |x1| <= 2^-8 |x|, |x2| <=
2^-17 |x|, and the sum is x itself.  Of the nine products of two floats they make the six largest; the rest, x1 y2 + x2 y1 + x2 y2, is at most
2^-24 |x y| and a little: U.  A wrong or missing x2 y0, x0 y2 or x1 y1 is an error of up to 128 U or 256 U, and of about 40 U and 90 U as a
root mean square: far more than one product's rounding, but little beside the bound of a sum of a hundred products.  So each number that is
looked at here is made of one product, or of products that have the same factor.

Bounds, in U relative to the sum of the terms' magnitudes.  A product: 1 for what is left out, 2 for the addition that brings in the largest of the
six (whether it rounds or cuts off), and less than 1/4 for the others, which are smaller by 2^8: PRODUCT = 3.25."""
import torch

U = 2.0 ** -24
PRODUCT = 3.25
# A logarithm, of one key, whose score is one product: that, the scale's conversion to units of log2, the maximum's rounding in them, the
# rounding of the sum with log2 of the probabilities' sum (1 each), the constant and the product of the way back (1 each); and, not relative,
# the exponential's two steps and log2's, 4.
LOGARITHM, LOGARITHM_ADDS = PRODUCT + 5, 4
# An output, of a few keys with the same value c: the products p c; each of them added with an error of 2 (two or four keys: 8, the six parts of
# each together); the probabilities' sum (4 additions and the two halves of a wave: 6), its reciprocal and the last product (2), joining of waves and of parts
# (4).
OUTPUT = PRODUCT + 8 + 6 + 2 + 4
# A probability of the backward pass, whose exponent is a small score (no error) less a logarithm of up to 1 in magnitude: the logarithm's conversion,
# 2 of up to 1.45, the sum's rounding, 1.45, and the exponential's two steps: 7.
PROBABILITY = 7
# dv, of one query with one key: the probability, the product with d_o; a part's sum and its joining add zeros.
VALUES = PROBABILITY + PRODUCT + 1
# dq and dk with o = 0, where d_o has one element: ds = p (d_o v), a product of two; times k or q, and the scale (a power of two).
QUERIES = PROBABILITY + PRODUCT + 1 + PRODUCT + 1
# (sums over the heads that share a key head add 2 for each)


def split(x):
    x = x.float()
    planes = []
    for _ in range(3):
        planes.append(x.to(torch.bfloat16).float())
        x = x - planes[-1]
    return planes


PAIRS = ((2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0))  # in the order in which they are added


def product(x, y, without=None):
    """x * y from their planes in 32 bits, or what comes out where one of the six is missing."""
    a, b, s = split(x), split(y), torch.zeros(torch.broadcast_shapes(x.shape, y.shape))
    for i, j in PAIRS:
        if (i, j) != without:
            s = s + a[i] * b[j]
    return s


def one_element(rows, heads, dim, generator, device, low=2.0, high=8.0):
    """(1, rows, heads, dim): a number of [low, high) or (-high, -low] in one element of each row, another one from row to row and from head to head."""
    x = torch.zeros(1, rows, heads, dim, device=device)
    r, h = torch.arange(rows, device=device)[:, None], torch.arange(heads, device=device)[None, :]
    value = torch.empty(rows, heads, device=device).uniform_(low, high, generator=generator)
    sign = torch.randint(0, 2, (rows, heads), generator=generator, device=device) * 2 - 1
    x[0, r, h, (r + 5 * h) % dim] = value * sign
    return x

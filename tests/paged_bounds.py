"""Error bounds of the paged attention that hold it to sums in round-to-nearest."""
import math


def sums_bound(size, weight, n, d, chain):
    """Error of fp32 rows that does not grow with n as a chain of truncated sums
    would.  Scores: each of the d products is off by 2^-22 of itself (rows in
    two f16), the d / 8 sums of tensor-core products by a unit 2^-23 each, the
    scales by 4 more: ds = (d / 8 + 6) 2^-23 max_t sum |q k| scale, a weight by
    a factor exp(+-2 ds).  16 units for the exponential, the weight's two f16
    and a step's own products; `chain` units where that many products are added
    on the tensor cores before a sum in round-to-nearest.  The sums themselves:
    the N additions of round-to-nearest are off by at most half a unit of the
    result each, in either direction; by Hoeffding their sum passes
    4 sqrt(N) halves once in 1500 times if each were off by all of it, and
    they are off by a third of that (a running sum is smaller than the result,
    a rounding smaller than half a unit).  N: n / 8 for the normaliser, n / 16
    for the weighted values."""
    ds = (d / 8 + 6) * 2.0 ** -23 * size
    return weight * (2 * ds + (16 + chain) * 2.0 ** -23 + 4 * 2.0 ** -24 * (math.sqrt(n / 8) + math.sqrt(n / 16)))

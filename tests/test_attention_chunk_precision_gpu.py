"""How exact chunk attention is beside its results' own rounding: weights of 16 bits, sums that do not lose with the length of the context.

Tolerances, relative to the value or to mass = sum p |v|.  A result's rounding to bf16 is half a step, 2^-8 at most.  A weight enters its
product with v as two bf16 numbers: 2^-8 of 2^-8 of it is left out, 2^-16.  The scores of these cases stay below 2^4 in powers of two and
their 128 products below 2^7: the tensor core cuts them eight times at 2^-17 each, 2^-14 in the sum and 2^-17 in the exponent after the
scale 1 / sqrt(128) log2 e = 2^-3; the exponent's own rounding and the exponential add 2^-19.  Sums of up to 600 positions lose 2^-23 of
themselves per MMA of eight per 64 positions at most, half of that on average over their growth: 2^-18.  In all less than 2^-15 of the mass,
twice (result and denominator): 2^-14."""
import numpy as np
import pytest
import torch

from test_attention_chunk_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,starts,heads", [([200, 33], [0, 350], (4, 2)), ([5, 9, 1], [500, 130, 63], (16, 8)), ([150] * 20, [37] * 20, (16, 8)), ([3], [590], (2, 1))])
def test_weights_keep_sixteen_bits(lens, starts, heads):
    c = Case(lens, starts, *heads, seed=11)
    d = c.run()
    want, tol, _, _ = c.expect()
    mass = (tol - 2.0 ** -8 * np.abs(want)) / (2.0 ** -8 + 2.0 ** -11)
    off = np.abs(d["out"].double().cpu().numpy() - want)
    bad = off > 2.0 ** -8 * np.abs(want) + 2.0 ** -14 * mass
    assert not bad.any(), f"{bad.sum()} of {bad.size}, the largest by {(off - 2.0 ** -8 * np.abs(want))[bad].max() / mass.max()}"

"""The stand-alone operators of include/csm_ops.h where they are used otherwise than in test_paged_ops.py: roundings of single steps, settings and
sizes at the end of their ranges, calls that have to be refused.  Tolerances count roundings (half a step: fp32 2^-24, bf16 2^-8)."""

import pytest
import torch

from csm_hf_amd import paged_prefix_attention
from test_paged_ops import BF16, Cache, DEV, HALF, attention64, check


# ---- attention -----------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("b,n_q,n_kv,hd,prefix,longest", [(40, 8, 2, 64, 900, 200), (130, 4, 1, 64, 300, 40), (40, 4, 2, 128, 900, 100), (9, 8, 2, 64, 700, 300)])
def test_attention_weights_of_decode_batches_are_not_rounded_to_bf16(b, n_q, n_kv, hd, prefix, longest):
    """One new token per sequence behind a shared prefix: beside the one rounding of the result, a weight is off by 2^-15 at most (a truncated bf16
    piece leaves less than 2^-7 of it, and of that the second piece is off by half a step)."""
    lens = [max(1, longest - (i * 37) % longest) for i in range(b)]
    cache = Cache(lens, 16, n_kv, hd, BF16, prefix=prefix, seed=b)
    q = torch.randn(b, n_q, hd, generator=torch.Generator().manual_seed(b)).to(BF16).to(DEV)
    got = paged_prefix_attention(q, *cache.args(), prefix_table=cache.prefix, prefix_len=prefix)
    want, tol = attention64(q, cache, lens, [1] * b, n_q, hd ** -0.5, False)
    mag, _ = attention64(q, _abs_v(cache), lens, [1] * b, n_q, hd ** -0.5, False)
    check(got, want, tol + mag * 2.0 ** -15 + want.abs() * HALF[BF16], 0.0)


def _abs_v(cache):
    other = object.__new__(Cache)
    other.__dict__.update(cache.__dict__, v=cache.v.abs())
    return other

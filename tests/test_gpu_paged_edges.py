"""The paged cache's operators on a B200 at the ends of their range: scores far apart, infinitely low ones, slots
without a sequence, outputs in the memory of inputs. Against float64, as in ``test_gpu_paged.py``."""
import numpy as np
import pytest
import torch

from paged_cases import UNIT, check, host, normal, offsets, oracle_rows

from moss_tts._runtime import kernels as K, native

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("slots", [4000, 40])
def test_blocks_taken_one_after_the_other_without_an_item(cuda_device, slots):
    """Few sequences among many empty ones: the answers to the requests for blocks follow at once on one another.
    Every call gives the same bits, the right ones, and no wait expires."""
    dev, d = cuda_device, 64
    real = [700, 1, 333]
    new = [0] * slots + [real[0]] + [0] * slots + [real[1], real[2]] + [0] * slots
    q, k, v = (normal(300 + i, sum(real), 8, d, device=dev) for i in range(3))
    cu = offsets(new, dev)
    native.error_word(clear=True)
    first = K.packed_attention(q, k, v, cu)
    outs = [K.packed_attention(q, k, v, cu) for _ in range(50)]
    assert native.error_word() == 0
    assert all(torch.equal(first, x) for x in outs)
    at = [0] + list(np.cumsum(real))
    hk, hv = host(k), host(v)
    want, bound = oracle_rows(q, lambda b: (hk[at[b]:at[b + 1]], hv[at[b]:at[b + 1]]), at, d ** -0.5, True, BF, UNIT[BF])
    check("padded batch, repeated", first, want, bound)

"""The paged cache's operators without a GPU: the float64 oracle against itself, and what the Python
wrappers and the C entry points refuse before anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as opaged
from paged_cases import host, ints, make_cache, normal, offsets

from moss_tts._runtime import kernels as K
from moss_tts._runtime import native

CPU = torch.device("cpu")


def test_oracle_gathers_pages_and_reads_missing_ones_as_zeros():
    lens = [37, 0, 64]
    kp, _, table = make_cache(1, lens, 2, 64, 16, torch.bfloat16, CPU)
    rows = normal(1 * 100 + 1, 48, 2, 64)  # sequence 0's, as make_cache draws them
    assert np.array_equal(opaged.gather(host(kp), host(table)[0], 37), host(rows)[:37])
    t = host(table).copy()
    t[0, 1] = -1
    got = opaged.gather(host(kp), t[0], 37)
    assert np.all(got[16:32] == 0) and np.array_equal(got[:16], host(rows)[:16])


def test_oracle_attention_is_softmax_of_what_a_row_sees():
    q, k, v = host(normal(2, 5, 4, 64)), host(normal(3, 3, 2, 64)), host(normal(4, 3, 2, 64))
    out, bound = opaged.attention(q, k, v, 0.125, True, 2.0 ** -8, 2.0 ** -8)
    assert np.all(out[:2] == 0) and np.all(bound[2:] > 0)  # 3 keys for 5 queries: the first two see none
    assert np.allclose(out[2, 0], v[0, 0])                 # one key: its value
    s = np.exp(0.125 * q[4, 3] @ k[:, 1].T)
    assert np.allclose(out[4, 3], (s / s.sum()) @ v[:, 1])


def test_oracle_rotation_keeps_the_norm():
    x = host(normal(5, 3, 64))
    angle = np.repeat(np.linspace(0, 3, 32)[None], 2, 0).reshape(-1)
    y = opaged.rotate(x, np.ones(64), np.cos(angle), np.sin(angle), 0.0)
    assert np.allclose((y ** 2).mean(-1), 1.0)


def _kv(**changes):
    kp, vp, table = make_cache(6, [20, 30], 2, 64, 16, torch.bfloat16, CPU)
    return {"k_pages": kp, "v_pages": vp, "page_table": table, "kv_lens": ints([20, 30])} | changes


@pytest.mark.parametrize("change", [
    {"k_pages": torch.zeros(3, 2, 24, 64, dtype=torch.bfloat16), "v_pages": torch.zeros(3, 2, 24, 64, dtype=torch.bfloat16)},
    {"k_pages": torch.zeros(3, 2, 16, 96, dtype=torch.bfloat16), "v_pages": torch.zeros(3, 2, 16, 96, dtype=torch.bfloat16)},
    {"k_pages": torch.zeros(3, 2, 16, 64)}, {"v_pages": torch.zeros(3, 2, 16, 64)},
    {"k_pages": torch.zeros(0, 2, 16, 64, dtype=torch.bfloat16), "v_pages": torch.zeros(0, 2, 16, 64, dtype=torch.bfloat16)},
    {"k_pages": torch.zeros(3, 2, 16, 68, dtype=torch.bfloat16)[..., :64], "v_pages": torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)},
    {"k_pages": torch.zeros(3, 1, 16, 64, dtype=torch.bfloat16).expand(3, 2, 16, 64), "v_pages": torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)},
    {"page_table": torch.zeros(2, 2)}, {"page_table": ints([0, 0])}, {"page_table": torch.zeros(0, 2, dtype=torch.int32)},
    {"page_table": torch.zeros(2, 0, dtype=torch.int32)}, {"kv_lens": ints([20])}, {"kv_lens": torch.tensor([20, 30])},
    {"kv_lens": ints([20, 0, 30, 0])[::2]},
])
def test_pages_are_checked(change):
    K._paged(**_kv(), dtype=torch.bfloat16, dev=-1)
    with pytest.raises(ValueError):
        K._paged(**_kv(**change), dtype=torch.bfloat16, dev=-1)  # -1: host tensors


def test_operators_refuse_host_tensors():
    kv = _kv()
    q = normal(7, 2, 4, 64)
    with pytest.raises(ValueError, match="no CPU path"):
        K.paged_attention_decode(q, *kv.values())
    with pytest.raises(ValueError, match="no CPU path"):
        K.paged_attention_prompt(q, *kv.values(), offsets([1, 1]))
    with pytest.raises(ValueError, match="no CPU path"):
        K.packed_attention(q, q, q, offsets([1, 1]))
    with pytest.raises(ValueError, match="no CPU path"):
        K.qk_rope_paged(q.view(2, -1), *[None] * 4, *kv.values(), None, 1e-6)


def test_entry_points_refuse_before_a_launch():
    """The C entry points' own checks, with addresses that nothing reads."""
    lib = native.library()
    P = 1 << 20  # 16-byte aligned, never dereferenced: each call fails a host check

    def kv(**c):
        f = dict(k=P, v=P, table=P, lens=P, ks=(4096, 1024, 64), vs=(4096, 1024, 64), trow=4, pages=3, heads=2, size=16,
                 d=64, most=4, batch=2, type=0) | c
        return native.PAGED_KV.pack(f["k"], f["v"], f["table"], f["lens"], *f["ks"], *f["vs"], f["trow"], f["pages"],
                                    f["heads"], f["size"], f["d"], f["most"], f["batch"], f["type"])

    assert native.PAGED_KV.size % 8 == 0 and native.PAGED_KV.size == 4 * 8 + 7 * 8 + 7 * 4 + 4
    bad_kv = [kv(**c) for c in (dict(k=0), dict(table=0), dict(k=P + 8), dict(ks=(4096, 1024, 60)), dict(ks=(0, 1024, 64)),
                                dict(vs=(4096, -8, 64)), dict(pages=0), dict(heads=0), dict(size=8), dict(size=48),
                                dict(size=512), dict(d=96), dict(most=0), dict(batch=0), dict(type=2), dict(lens=P + 2))]
    for x in bad_kv:
        assert lib.mt_paged_attention_decode(P, 256, 64, x, 4, 0.1, P, P, None, 0, None) == 1
        assert lib.mt_paged_attention_prompt(P, 256, 64, x, P, 2, 4, 0.1, P, None, None, 0, None) == 1
        assert lib.mt_qk_rope_paged(P, P, P, P, P, 64, 0, x, P, 2, 4, 512, P, 1e-6, None, 0, None) == 1
    good = kv()
    for a in ((None, 256, 64, good, 4, 0.1, P), (P, 256, 64, good, 3, 0.1, P), (P, 256, 64, good, 0, 0.1, P),
              (P, 256, 64, good, 130, 0.1, P), (P, 250, 64, good, 4, 0.1, P), (P, 256, 64, good, 4, 0.1, P + 4),
              (P, 256, 64, None, 4, 0.1, P)):
        assert lib.mt_paged_attention_decode(*a, P, None, 0, None) == 1
    assert lib.mt_paged_attention_decode(P, 256, 64, good, 4, 0.1, P, None, None, 0, None) == 1  # no workspace
    for a in ((P, 256, 64, P, 128, 64, P, 128, 64, P, P, 0), (P, 256, 64, P, 128, 60, P, 128, 64, P, P, 1),
              (P, 256, 64, P, 128, 64, P, 0, 64, P, P, 1), (P, 256, 64, P, 128, 64, P, 128, 64, None, P, 1)):
        assert lib.mt_packed_attention(*a, 4, 4, 4, 2, 64, 0, 1, 0.1, P, None, 0, None) == 1
    for c in (dict(tokens=0), dict(cu=None, tokens=3), dict(row=504), dict(rows=0), dict(qkv=P + 2), dict(nq=0)):
        f = dict(qkv=P, rows=64, cu=P, tokens=2, nq=4, row=512) | c
        assert lib.mt_qk_rope_paged(f["qkv"], P, P, P, P, f["rows"], 0, good, f["cu"], f["tokens"], f["nq"], f["row"], P,
                                    1e-6, None, 0, None) == 1
    assert isinstance(good, bytes) and ctypes.sizeof(ctypes.c_void_p) == 8

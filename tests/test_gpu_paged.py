"""The paged key-value cache on a B200: write of new tokens, decode attention, packed and paged prompt
attention, against float64 and within the bounds that ``oracle/paged.py`` derives. Rows that no sequence
holds are NaN and unused page-table entries lie outside the cache, in every case."""
import numpy as np
import pytest
import torch

from oracle import paged as opaged
from paged_cases import UNIT, check, host, ints, make_cache, normal, offsets, oracle_rows

from moss_tts._runtime import kernels as K, native
from moss_tts._runtime.engine import rope_tables

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
DECODE_WEIGHT = 2.0 ** -15  # decode keeps softmax weights to 16 bits or more
EPS = 1e-6


# ------------------------------------------------------------------------------------ write
def _write_inputs(dev, seed, new, lens, nq, nkv, d, page, dtype, table_dtype, pad=0):
    tokens = sum(new) + pad
    qkv = normal(seed, tokens, (nq + 2 * nkv) * d, dtype=dtype, device=dev)
    qw = (1 + 0.1 * normal(seed + 1, d, dtype=torch.float32)).to(dtype).to(dev)
    kw = (1 + 0.1 * normal(seed + 2, d, dtype=torch.float32)).to(dtype).to(dev)
    cos, sin = rope_tables(max(lens), d)
    cos, sin = (t.to(table_dtype).to(dev) for t in (cos, sin))
    return qkv, qw, kw, cos, sin


def _expect_write(qkv, qw, kw, cos, sin, kp, vp, table, lens, cu, nq, nkv, d):
    """Float64 results and bounds: the rounding at the store and 16 fp32 roundings of |y cos| + |y' sin|."""
    page = kp.shape[2]
    x = host(qkv).reshape(-1, nq + 2 * nkv, d)
    q, k, v = np.full((x.shape[0], nq, d), 7.0), host(kp), host(vp)
    qb, kb = np.zeros_like(q), np.zeros_like(k)
    unit = UNIT[qkv.dtype]
    for t, b, pos in opaged.sequence_rows(cu, x.shape[0], lens):
        c, s = host(cos)[pos], host(sin)[pos]
        for heads, w, res, lim, at in ((slice(0, nq), qw, q, qb, t), (slice(nq, nq + nkv), kw, k, kb, None)):
            y = opaged.rotate(x[t, heads], host(w), c, s, EPS)
            near = np.abs(opaged.rotate(x[t, heads], host(w), np.ones(d), np.zeros(d), EPS))
            size = near * np.abs(c) + np.roll(near, d // 2, -1) * np.abs(s)
            bound = unit * np.abs(y) + 16 * 2.0 ** -24 * size + 2.0 ** -25
            if at is None:
                res[int(table[b, pos // page]), :, pos % page] = y
                lim[int(table[b, pos // page]), :, pos % page] = bound
            else:
                res[at], lim[at] = y, bound
        v[int(table[b, pos // page]), :, pos % page] = x[t, nq + nkv:]
    return q, qb, k, kb, v


def _same_or_near(label, got, want, bound):
    """Within the bound where there is one, else the same, NaN included."""
    got = host(got).reshape(want.shape)
    assert np.array_equal(got[bound == 0], want[bound == 0], equal_nan=True), label
    check(label, torch.from_numpy(np.where(bound > 0, got, 0.0)), np.where(bound > 0, want, 0.0), bound)


@pytest.mark.parametrize("dtype,table_dtype,nq,nkv,d,page,new,past,pad", [
    (BF, BF, 32, 8, 128, 64, [1, 1, 1], [0, 63, 64], 0),
    (BF, torch.float32, 4, 1, 128, 16, [5, 0, 37, 1], [0, 20, 15, 300], 3),
    (HF, HF, 6, 2, 64, 32, [33, 2, 64], [31, 0, 1], 5),
    (HF, torch.float32, 3, 3, 64, 256, [300], [0], 0),
    (BF, BF, 7, 1, 64, 128, [1] * 70, list(range(70)), 2),
])
@pytest.mark.parametrize("order", ["heads", "rows"])
def test_write_matches_float64_and_touches_nothing_else(cuda_device, dtype, table_dtype, nq, nkv, d, page, new, past, pad, order):
    dev = cuda_device
    lens = [n + p for n, p in zip(new, past)]
    kp, vp, table = make_cache(3, lens, nkv, d, page, dtype, dev, order=order)
    qkv, qw, kw, cos, sin = _write_inputs(dev, 11, new, lens, nq, nkv, d, page, dtype, table_dtype, pad)
    cu = offsets(new, dev)
    out = torch.full((qkv.shape[0], nq, d), 7.0, device=dev, dtype=dtype)
    q, qb, k, kb, v = _expect_write(qkv, qw, kw, cos, sin, kp, vp, host(table), lens, host(cu).astype(int), nq, nkv, d)
    status = ints([0], dev)
    got = K.qk_rope_paged(qkv, qw, kw, cos, sin, kp, vp, table, ints(lens, dev), cu, EPS, out=out, status=status)
    assert got is out and int(status.item()) == 0
    _same_or_near("q", got, q, qb)
    _same_or_near("k pages", kp, k, kb)
    assert np.array_equal(host(vp), v, equal_nan=True)  # values are copied; every other row is as it was


def test_write_of_one_token_each_needs_no_offsets(cuda_device):
    dev, nq, nkv, d = cuda_device, 8, 2, 128
    lens = [1, 64, 65, 200]
    kp, vp, table = make_cache(4, lens, nkv, d, 64, BF, dev)
    qkv, qw, kw, cos, sin = _write_inputs(dev, 12, [1] * 4, lens, nq, nkv, d, 64, BF, BF)
    wide = torch.full((4, qkv.shape[1] + 64), 9.0, device=dev, dtype=BF)
    wide[:, :qkv.shape[1]] = qkv
    a = (kp.clone(), vp.clone())
    q1 = K.qk_rope_paged(qkv, qw, kw, cos, sin, kp, vp, table, ints(lens, dev), offsets([1] * 4, dev), EPS)
    q2 = K.qk_rope_paged(wide[:, :qkv.shape[1]], qw, kw, cos, sin, *a, table, ints(lens, dev), None, EPS)
    assert torch.equal(q1, q2)
    assert torch.equal(kp.nan_to_num(9.0), a[0].nan_to_num(9.0)) and torch.equal(vp.nan_to_num(9.0), a[1].nan_to_num(9.0))


def test_write_outside_the_tables_writes_nothing_and_says_so(cuda_device):
    dev, nq, nkv, d = cuda_device, 4, 2, 128
    lens = [40, 40]
    kp, vp, table = make_cache(5, lens, nkv, d, 16, BF, dev, rubbish=0.5)
    qkv, qw, kw, cos, sin = _write_inputs(dev, 13, [1, 1], lens, nq, nkv, d, 16, BF, BF)
    before = kp.clone(), vp.clone()
    for lens_now, bad_page, want in (([49, 0], None, 1), ([41, 41], None, 1), ([40, 40], -1, 3), ([40, 40], 1 << 20, 3)):
        t = table.clone()
        if bad_page is not None:
            t[:] = bad_page
        status = ints([0], dev)
        K.qk_rope_paged(qkv, qw, kw, cos, sin, kp, vp, t, ints(lens_now, dev), None, EPS, status=status)
        assert int(status.item()) == want
        assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])


# ------------------------------------------------------------------------------------ decode
def _decode(dev, seed, lens, nq, nkv, d, page, dtype, order="heads", scale=None, heavy=1.0):
    kp, vp, table = make_cache(seed, lens, nkv, d, page, dtype, dev, order=order)
    q = normal(seed + 50, len(lens), nq, d, dtype=dtype, device=dev) * heavy
    status = ints([0], dev)
    out = K.paged_attention_decode(q, kp, vp, table, ints(lens, dev), scale=scale, status=status)
    assert int(status.item()) == 0
    hk, hv, ht = host(kp), host(vp), host(table)
    want, bound = oracle_rows(q, lambda b: (opaged.gather(hk, ht[b], lens[b]), opaged.gather(hv, ht[b], lens[b])),
                              list(range(len(lens) + 1)), d ** -0.5 if scale is None else scale, True, dtype, DECODE_WEIGHT)
    check(f"decode {dtype} {nq}/{nkv}x{d} page {page}", out, want, bound)
    return out


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nq,nkv,d,page", [(32, 8, 128, 64), (4, 1, 128, 16), (7, 1, 64, 32), (3, 3, 128, 256),
                                           (24, 8, 64, 128), (16, 1, 128, 64), (64, 1, 64, 16), (13, 1, 128, 128)])
def test_decode_lengths_and_heads(cuda_device, dtype, nq, nkv, d, page):
    _decode(cuda_device, 21, [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500], nq, nkv, d, page, dtype)


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [5000], [1, 4097, 0, 300], [33] * 300])
@pytest.mark.parametrize("order", ["heads", "rows"])
def test_decode_splits_and_batches(cuda_device, lens, order):
    _decode(cuda_device, 22, lens, 8, 2, 128, 64, BF, order=order)


def test_decode_of_sharp_and_flat_scores(cuda_device):
    _decode(cuda_device, 23, [700, 64, 1], 8, 2, 128, 32, BF, heavy=20.0)  # one key takes nearly all
    _decode(cuda_device, 24, [700, 64, 1], 8, 2, 64, 32, HF, scale=0.0)     # the mean of the values
    _decode(cuda_device, 25, [700, 64, 1], 8, 2, 64, 32, HF, scale=-0.3)


def test_decode_far_pages_pass_32_bit_offsets(cuda_device):
    dev, nkv, page, d = cuda_device, 8, 256, 128
    count = (1 << 31) // (nkv * page * d) + 40  # over 2^31 elements: 2^32 bytes and more
    kp = torch.empty(count, nkv, page, d, device=dev, dtype=BF)
    vp = torch.empty(count, nkv, page, d, device=dev, dtype=BF)
    ids = [count - 1, 0, count - 7]
    for i, pid in enumerate(ids):
        kp[pid], vp[pid] = (normal(30 + 2 * i + j, nkv, page, d, device=dev) for j in range(2))
    table, length = ints([ids], dev), 600
    q = normal(40, 1, 32, d, device=dev)
    out = K.paged_attention_decode(q, kp, vp, table, ints([length], dev))
    small = [torch.stack([p[i] for i in ids]) for p in (kp, vp)]
    hk, hv = (opaged.gather(host(p), [0, 1, 2], length) for p in small)
    want, bound = oracle_rows(q, lambda b: (hk, hv), [0, 1], d ** -0.5, True, BF, DECODE_WEIGHT)
    check("far pages", out, want, bound)
    prompt = K.paged_attention_prompt(q, kp, vp, table, ints([length], dev), offsets([1], dev))
    want, bound = oracle_rows(q, lambda b: (hk, hv), [0, 1], d ** -0.5, True, BF, UNIT[BF])
    check("far pages, prompt form", prompt, want, bound)
    qkv = normal(41, 1, (32 + 16) * d, device=dev)
    w = torch.ones(d, device=dev, dtype=BF)
    cos, sin = (t.to(dev) for t in rope_tables(length, d))
    K.qk_rope_paged(qkv, w, w, cos, sin, kp, vp, table, ints([length], dev), None, EPS)
    pos = length - 1
    assert torch.equal(vp[ids[pos // page], :, pos % page].reshape(-1), qkv[0, (32 + 8) * d:])


@pytest.mark.parametrize("op", ["decode", "prompt"])
def test_bad_pages_read_as_zeros_and_bad_lengths_are_cut(cuda_device, op):
    dev, nq, nkv, d, page = cuda_device, 8, 2, 128, 16
    lens = [100, 100]
    kp, vp, table = make_cache(26, lens, nkv, d, page, BF, dev)
    q = normal(27, 2, nq, d, device=dev)
    hk, hv = host(kp), host(vp)
    for bad, lens_now, code in ((-1, [100, 100], 3), (1 << 29, [100, 70], 3), (None, [1 << 20, 100], 1)):
        t = table.clone()
        if bad is not None:
            t[0, 2] = bad
        status = ints([0], dev)
        args = q, kp, vp, t, ints(lens_now, dev)
        if bad is None:  # 7 pages of 16 hold 112 rows; rows 100 and on are NaN: give them values first
            last = int(table[0, 6])
            kp[last, :, 4:], vp[last, :, 4:] = 0.25, 0.5
            hk, hv = host(kp), host(vp)
        out = (K.paged_attention_decode(*args, status=status) if op == "decode"
               else K.paged_attention_prompt(*args, offsets([1, 1], dev), status=status))
        assert int(status.item()) == code
        ht, real = host(t), [min(n, 112) for n in lens_now]
        want, bound = oracle_rows(q, lambda b: (opaged.gather(hk, ht[b], real[b]), opaged.gather(hv, ht[b], real[b])),
                                  [0, 1, 2], d ** -0.5, True, BF, DECODE_WEIGHT if op == "decode" else UNIT[BF])
        check(f"{op}, bad {bad}", out, want, bound)


# ------------------------------------------------------------------------------------ prompts
def _packed(dev, seed, new, lens, nq, nkv, d, dtype, causal=True, pad=0, scale=None):
    tokens = sum(new) + pad
    q = normal(seed, max(tokens, 1), nq, d, dtype=dtype, device=dev)
    k, v = (normal(seed + i, sum(lens) + pad + 1, nkv, d, dtype=dtype, device=dev) for i in (1, 2))
    q[sum(new):], k[sum(lens):], v[sum(lens):] = float("nan"), float("nan"), float("nan")
    out = torch.full_like(q, 7.0)
    got = K.packed_attention(q, k, v, offsets(new, dev), offsets(lens, dev), causal=causal, scale=scale, out=out)
    assert got is out
    starts = np.concatenate(([0], np.cumsum(lens)))
    hk, hv = host(k), host(v)
    want, bound = oracle_rows(q[:sum(new)], lambda b: (hk[starts[b]:starts[b + 1]], hv[starts[b]:starts[b + 1]]),
                              np.concatenate(([0], np.cumsum(new))), d ** -0.5 if scale is None else scale, causal, dtype,
                              UNIT[dtype])
    check(f"packed {dtype} {nq}/{nkv}x{d} causal {causal}", got[:sum(new)], want, bound)
    assert bool((got[sum(new):] == 7.0).all())  # rows behind the last sequence


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 128), (3, 3, 64), (7, 1, 128), (8, 1, 64), (64, 1, 128), (2, 2, 128), (5, 1, 64),
                                      (24, 2, 128)])
def test_packed_heads_and_lengths(cuda_device, dtype, nq, nkv, d):
    new = [1, 0, 17, 64, 65, 130, 2]
    _packed(cuda_device, 60, new, new, nq, nkv, d, dtype, pad=3)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,lens", [
    ([5, 40, 0, 3, 128], [700, 40, 30, 0, 129]),   # keys from before, none new, no key at all
    ([40, 200, 3], [10, 1, 3]),                    # fewer keys than queries: the first rows see none
    ([1], [1]), ([1], [0]), ([127], [128]), ([129], [257]), ([300], [385]),
    ([1] * 200, list(range(200))),
])
def test_packed_queries_and_keys_of_other_lengths(cuda_device, new, lens, causal):
    _packed(cuda_device, 61, new, lens, 4, 1, 128, BF, causal=causal)
    _packed(cuda_device, 62, new, lens, 4, 2, 64, HF, causal=causal, pad=2)


def test_packed_long_prompt(cuda_device):
    _packed(cuda_device, 63, [1500], [1500], 4, 1, 128, BF)
    _packed(cuda_device, 64, [64], [5001], 4, 1, 128, BF)


def test_packed_scales(cuda_device):
    _packed(cuda_device, 65, [200, 70], [200, 70], 4, 1, 128, BF, scale=2.0)  # sharp
    _packed(cuda_device, 66, [200, 70], [200, 70], 4, 1, 64, HF, scale=0.0)
    _packed(cuda_device, 67, [200, 70], [200, 70], 4, 1, 128, BF, scale=-0.05)


def test_packed_rising_scores_move_the_running_maximum(cuda_device):
    """Scores that grow along the keys by hundreds: the running maximum moves at every tile."""
    dev, n, d = cuda_device, 700, 128
    q = torch.ones(n, 2, d, device=dev, dtype=BF)
    k = (torch.arange(n, device=dev)[:, None, None] * 0.125).expand(n, 2, d).to(BF).contiguous()
    v = normal(70, n, 2, d, device=dev)
    for sign in (1, -1):
        got = K.packed_attention(q, k * sign, v, offsets([n], dev))
        want, bound = oracle_rows(q, lambda b: (host(k) * sign, host(v)), [0, n], d ** -0.5, True, BF, UNIT[BF])
        check(f"rising by {sign}", got, want, bound)


@pytest.mark.parametrize("dtype,d", [(BF, 64), (HF, 64), (HF, 128)])
@pytest.mark.parametrize("step", [0.125, 0.02, -0.125])
def test_packed_rising_scores_in_either_type(cuda_device, dtype, d, step):
    """Steps whose weights leave fp16's range, or the reference's, by little and by far."""
    dev, n = cuda_device, 500
    q = torch.ones(n, 2, d, device=dev, dtype=dtype)
    k = (torch.arange(n, device=dev)[:, None, None] * step).expand(n, 2, d).to(dtype).contiguous()
    v = normal(75, n, 2, d, dtype=dtype, device=dev)
    got = K.packed_attention(q, k, v, offsets([n], dev))
    want, bound = oracle_rows(q, lambda b: (host(k), host(v)), [0, n], d ** -0.5, True, dtype, UNIT[dtype])
    check(f"rising by {step} {dtype}", got, want, bound)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("first", [12.0, -12.0])
def test_packed_first_key_far_from_the_others(cuda_device, dtype, first):
    """The reference starts at the first key's score: here scores of +-136 beside some of +-10."""
    dev, n, d = cuda_device, 300, 128
    q = torch.ones(n, 2, d, device=dev, dtype=dtype)
    k = normal(76, n, 2, d, dtype=dtype, device=dev)
    k[0] = first
    v = normal(77, n, 2, d, dtype=dtype, device=dev)
    got = K.packed_attention(q, k, v, offsets([n], dev))
    want, bound = oracle_rows(q, lambda b: (host(k), host(v)), [0, n], d ** -0.5, True, dtype, UNIT[dtype])
    check(f"first key {first} {dtype}", got, want, bound)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rise", [30.0, 80.0, 87.3, 88.0, 95.0])
@pytest.mark.parametrize("keys", [100, 300, 3000])
def test_packed_weights_near_the_end_of_their_range(cuda_device, dtype, rise, keys):
    """The first key's score is 0, the others lie `rise` above it: beside it their weights add up to up to
    fp32's largest number and beyond, with values so small that their products do not."""
    dev, d, n = cuda_device, 64, 40
    q = torch.zeros(n, 16, d, device=dev, dtype=dtype)
    q[..., 0] = 1
    k = torch.zeros(keys, 1, d, device=dev, dtype=dtype)
    k[1:, 0, 0] = 1
    v = normal(83, keys, 1, d, dtype=torch.float32).mul(0.01).to(dtype).to(dev)
    got = K.packed_attention(q, k, v, offsets([n], dev), offsets([keys], dev), scale=rise)
    want, bound = oracle_rows(q, lambda b: (host(k), host(v)), [0, n], rise, True, dtype, UNIT[dtype])
    check(f"rise of {rise} over {keys} keys {dtype}", got, want, bound)


def test_packed_many_short_sequences(cuda_device):
    """More items than CTAs, taken on demand, among them empty sequences."""
    r = np.random.default_rng(78)
    new = [int(x) for x in r.integers(0, 30, 900)]
    _packed(cuda_device, 79, new, [n + int(x) for n, x in zip(new, r.integers(0, 40, 900))], 4, 2, 64, BF, pad=5)
    _packed(cuda_device, 79, new[:300], new[:300], 6, 3, 128, HF)


@pytest.mark.parametrize("dtype,nq,nkv,d", [(BF, 4, 1, 128), (HF, 6, 2, 64), (BF, 14, 2, 64), (HF, 8, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_few_rows_over_many_keys_are_cut_and_joined(cuda_device, dtype, nq, nkv, d, causal):
    _packed(cuda_device, 200, [48], [4097], nq, nkv, d, dtype, causal=causal, pad=2)
    _packed(cuda_device, 201, [1, 0, 3], [2500, 700, 0], nq, nkv, d, dtype, causal=causal)
    _packed(cuda_device, 202, [40, 2], [30, 1700], nq, nkv, d, dtype, causal=causal)  # rows without a key


def test_cut_prompts_over_pages(cuda_device):
    dev, nq, nkv, d, page = cuda_device, 8, 2, 128, 32
    new, lens = [20, 1, 0], [3000, 900, 10]
    kp, vp, table = make_cache(210, lens, nkv, d, page, BF, dev)
    q = normal(211, sum(new), nq, d, device=dev)
    hk, hv, ht = host(kp), host(vp), host(table)
    for bad in (False, True):
        t, status = table.clone(), ints([0], dev)
        if bad:
            t[0, 40], ht[0, 40] = 1 << 28, -1
        out = K.paged_attention_prompt(q, kp, vp, t, ints(lens, dev), offsets(new, dev), status=status)
        assert int(status.item()) == (3 if bad else 0)
        want, bound = oracle_rows(q, lambda b: (opaged.gather(hk, ht[b], lens[b]), opaged.gather(hv, ht[b], lens[b])),
                                  [0, 20, 21, 21], d ** -0.5, True, BF, UNIT[BF])
        check(f"cut over pages, bad {bad}", out, want, bound)


def test_packed_takes_slices_of_one_projection(cuda_device):
    dev, nq, nkv, d, new = cuda_device, 8, 2, 128, [70, 9, 200]
    qkv = normal(71, sum(new), nq + 2 * nkv, d, device=dev)
    q, k, v = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
    a = K.packed_attention(q, k, v, offsets(new, dev))
    b = K.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), offsets(new, dev), offsets(new, dev))
    assert torch.equal(a, b)
    t = torch.empty(nq, sum(new), d, device=dev, dtype=BF).transpose(0, 1)  # heads outermost
    t.copy_(q)
    assert torch.equal(a, K.packed_attention(t, k, v, offsets(new, dev)))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_may_not_see_does_not_reach_it(cuda_device, bad):
    """Non-finite keys and values of the sequence beside, and behind a row in its own sequence."""
    dev, nq, nkv, d, new = cuda_device, 8, 2, 128, [100, 60, 150]
    q = normal(72, sum(new), nq, d, device=dev)
    k, v = normal(73, sum(new), nkv, d, device=dev), normal(74, sum(new), nkv, d, device=dev)
    clean = K.packed_attention(q, k, v, offsets(new, dev))
    for at in (100, 159, 40, 200):
        kb, vb = k.clone(), v.clone()
        kb[at], vb[at] = bad, bad
        for kk, vv in ((kb, v), (k, vb), (kb, vb)):
            got = K.packed_attention(q, kk, vv, offsets(new, dev))
            first, last = max(s for s in (0, 100, 160) if s <= at), min(e for e in (100, 160, 310) if e > at)
            same = [i for i in range(sum(new)) if not at <= i < last]
            assert torch.isfinite(got[same]).all(), (bad, at)
            err = (got[same].double() - clean[same].double()).abs()
            assert bool((err <= 4 * UNIT[BF] * clean[same].double().abs() + 4 * UNIT[BF]).all())
            if vv is vb:  # and the rows that see the value have it
                assert not torch.isfinite(got[at:last]).all(-1).any()
            assert first <= at


def test_what_a_row_may_not_see_does_not_reach_it_in_cut_items(cuda_device):
    dev, nq, nkv, d, n, m = cuda_device, 4, 1, 128, 40, 3000
    q = normal(220, n, nq, d, device=dev)
    k, v = normal(221, m, nkv, d, device=dev), normal(222, m, nkv, d, device=dev)
    clean = K.packed_attention(q, k, v, offsets([n], dev), offsets([m], dev))
    for at in (m - 1, m - 20, 100):
        vb = v.clone()
        vb[at] = float("nan")
        got = K.packed_attention(q, k, vb, offsets([n], dev), offsets([m], dev))
        sees = torch.arange(n, device=dev) + m - n >= at
        assert torch.isnan(got[sees]).all() and torch.isfinite(got[~sees]).all()
        err = (got[~sees].double() - clean[~sees].double()).abs()
        assert bool((err <= 4 * UNIT[BF] * clean[~sees].double().abs() + 4 * UNIT[BF]).all())


def test_scores_that_are_not_finite_reach_the_rows_that_see_them(cuda_device):
    dev, d = cuda_device, 128
    for dtype in (BF, HF):
        q = normal(230, 200, 2, d, dtype=dtype, device=dev)
        k, v = normal(231, 200, 2, d, dtype=dtype, device=dev), normal(232, 200, 2, d, dtype=dtype, device=dev)
        k[150, 1] = float("nan")
        q[20, 0] = float("nan")
        got = K.packed_attention(q, k, v, offsets([200], dev))
        bad = torch.zeros(200, 2, dtype=torch.bool, device=dev)
        bad[150:, 1] = True
        bad[20, 0] = True
        assert torch.equal(torch.isnan(got).all(-1), bad) and torch.equal(torch.isnan(got).any(-1), bad)
        out = K.paged_attention_decode(q[19:21], k[:, None].transpose(0, 1).reshape(1, 200, 2, d)[:, :192].transpose(1, 2)
                                       .reshape(1, 2, 6, 32, d).transpose(1, 2)[0].contiguous(),
                                       v[:192].transpose(0, 1).reshape(2, 6, 32, d).transpose(0, 1).contiguous(),
                                       ints([list(range(6))] * 2, dev), ints([192, 192], dev))
        want = torch.tensor([[False, True], [True, True]], device=dev)
        assert torch.equal(torch.isnan(out).all(-1), want) and torch.equal(torch.isnan(out).any(-1), want)


@pytest.mark.parametrize("dtype,nq,nkv,d,page", [(BF, 8, 2, 128, 16), (BF, 4, 1, 128, 64), (HF, 6, 2, 64, 32),
                                                 (HF, 7, 1, 128, 256), (BF, 3, 3, 64, 128)])
@pytest.mark.parametrize("order", ["heads", "rows"])
def test_prompt_over_pages(cuda_device, dtype, nq, nkv, d, page, order):
    dev = cuda_device
    new, past = [1, 40, 0, 130, 64, 7], [0, 0, 20, 200, 65, 600]
    lens = [n + p for n, p in zip(new, past)]
    kp, vp, table = make_cache(80, lens, nkv, d, page, dtype, dev, order=order)
    q = normal(81, sum(new) + 4, nq, d, dtype=dtype, device=dev)
    out, status = torch.full_like(q, 7.0), ints([0], dev)
    K.paged_attention_prompt(q, kp, vp, table, ints(lens, dev), offsets(new, dev), out=out, status=status)
    assert int(status.item()) == 0 and bool((out[sum(new):] == 7.0).all())
    hk, hv, ht = host(kp), host(vp), host(table)
    want, bound = oracle_rows(q[:sum(new)], lambda b: (opaged.gather(hk, ht[b], lens[b]), opaged.gather(hv, ht[b], lens[b])),
                              np.concatenate(([0], np.cumsum(new))), d ** -0.5, True, dtype, UNIT[dtype])
    check(f"prompt over pages {dtype} {nq}/{nkv}x{d} page {page}", out[:sum(new)], want, bound)


# ------------------------------------------------------------------------------------ together
def test_a_single_token_is_as_exact_by_either_entry_point(cuda_device):
    """One new token through the prompt entry points is held to the decode kernel's bound."""
    dev = cuda_device
    for dtype, nq, nkv, d, lens in ((BF, 8, 2, 128, [1000, 3, 129]), (HF, 7, 1, 64, [2000]), (HF, 4, 1, 128, [64, 65]),
                                    (BF, 3, 3, 64, [500] * 8)):
        kp, vp, table = make_cache(250, lens, nkv, d, 64, dtype, dev)
        q = normal(251, len(lens), nq, d, dtype=dtype, device=dev)
        ln, cu = ints(lens, dev), offsets([1] * len(lens), dev)
        hk, hv, ht = host(kp), host(vp), host(table)
        want, bound = oracle_rows(q, lambda b: (opaged.gather(hk, ht[b], lens[b]), opaged.gather(hv, ht[b], lens[b])),
                                  list(range(len(lens) + 1)), d ** -0.5, True, dtype, DECODE_WEIGHT)
        check("decode", K.paged_attention_decode(q, kp, vp, table, ln), want, bound)
        check("prompt", K.paged_attention_prompt(q, kp, vp, table, ln, cu), want, bound)
        packed = [torch.cat([torch.from_numpy(opaged.gather(x, ht[b], lens[b])) for b in range(len(lens))]).to(dtype).to(dev)
                  for x in (hk, hv)]
        check("packed", K.packed_attention(q, *packed, cu, offsets(lens, dev)), want, bound)


def test_prompts_then_steps_through_one_cache(cuda_device):
    """Prompts in two chunks, then decode steps, through the pages: each attention result against the
    whole sequence in float64, from the rotated rows that the writes stored."""
    dev, nq, nkv, d, page = cuda_device, 8, 2, 128, 16
    prompt, steps = [37, 1, 90], 5
    full = [n + steps for n in prompt]
    kp, vp, table = make_cache(90, full, nkv, d, page, BF, dev)
    kp.fill_(float("nan"))
    vp.fill_(float("nan"))
    qw = (1 + 0.1 * normal(91, d, dtype=torch.float32)).to(BF).to(dev)
    kw = (1 + 0.1 * normal(92, d, dtype=torch.float32)).to(BF).to(dev)
    cos, sin = (t.to(dev) for t in rope_tables(max(full), d))
    first = [20, 1, 64]
    chunks = [first, [n - f for n, f in zip(prompt, first)]] + [[1] * 3] * steps
    lens = [0, 0, 0]
    for i, new in enumerate(chunks):
        lens = [n + m for n, m in zip(lens, new)]
        qkv = normal(93 + i, sum(new), (nq + 2 * nkv) * d, device=dev)
        cu, now = offsets(new, dev), ints(lens, dev)
        q = K.qk_rope_paged(qkv, qw, kw, cos, sin, kp, vp, table, now, cu, EPS)
        step = i >= 2
        got = (K.paged_attention_decode(q, kp, vp, table, now) if step
               else K.paged_attention_prompt(q, kp, vp, table, now, cu))
        hk, hv, ht = host(kp), host(vp), host(table)
        want, bound = oracle_rows(q, lambda b: (opaged.gather(hk, ht[b], lens[b]), opaged.gather(hv, ht[b], lens[b])),
                                  host(cu).astype(int), d ** -0.5, True, BF, DECODE_WEIGHT if step else UNIT[BF])
        check(f"call {i}", got, want, bound)
        # the last value rows are this call's
        for b, n in enumerate(new):
            if n:
                row = host(qkv)[host(cu).astype(int)[b + 1] - 1].reshape(-1, d)[nq + nkv:]
                assert np.array_equal(opaged.gather(hv, ht[b], lens[b])[-1], row)


def test_two_graphs_and_two_streams_at_once(cuda_device):
    """Captured once, replayed at once on two streams with other inputs: neither touches the other's."""
    dev, nq, nkv, d, page = cuda_device, 8, 2, 128, 64
    lens, new = [3000, 500, 64], [40, 100, 1]
    sides = []
    for side in range(2):
        kp, vp, table = make_cache(110 + side, lens, nkv, d, page, BF, dev)
        q = normal(120 + side, 3, nq, d, device=dev)
        qp = normal(130 + side, sum(new), nq, d, device=dev)
        ln, cu = ints(lens, dev), offsets(new, dev)
        plain = [K.paged_attention_decode(q, kp, vp, table, ln), K.paged_attention_prompt(qp, kp, vp, table, ln, cu)]
        out, outp, stream, graph = torch.zeros_like(q), torch.zeros_like(qp), torch.cuda.Stream(dev), torch.cuda.CUDAGraph()
        torch.cuda.synchronize(dev)
        with torch.cuda.graph(graph, stream=stream):
            K.paged_attention_decode(q, kp, vp, table, ln, out=out)
            K.paged_attention_prompt(qp, kp, vp, table, ln, cu, out=outp)
        sides.append((plain, out, outp, stream, graph, (q, qp, kp, vp, table, ln, cu)))
    torch.cuda.synchronize(dev)
    for _ in range(5):
        for plain, out, outp, stream, graph, _ in sides:
            with torch.cuda.stream(stream):
                out.zero_()
                outp.zero_()
                graph.replay()
    torch.cuda.synchronize(dev)
    for plain, out, outp, *_ in sides:
        assert torch.equal(plain[0], out) and torch.equal(plain[1], outp)


def test_same_inputs_give_the_same_bits(cuda_device):
    dev = cuda_device
    kp, vp, table = make_cache(140, [4000, 77], 2, 128, 64, BF, dev)
    q, qp = normal(141, 2, 8, 128, device=dev), normal(142, 120, 8, 128, device=dev)
    ln, cu = ints([4000, 77], dev), offsets([60, 60], dev)
    a = K.paged_attention_decode(q, kp, vp, table, ln), K.paged_attention_prompt(qp, kp, vp, table, ln, cu)
    for _ in range(5):
        b = K.paged_attention_decode(q, kp, vp, table, ln), K.paged_attention_prompt(qp, kp, vp, table, ln, cu)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_long_context_many_calls_in_a_row(cuda_device):
    """Dozens of chunks a CTA, calls queued without a wait between them: the chunks' copies land in any order."""
    dev = cuda_device
    kp, vp, table = make_cache(145, [32749], 8, 128, 128, BF, dev)
    q, ln = normal(146, 1, 32, 128, device=dev), ints([32749], dev)
    first = K.paged_attention_decode(q, kp, vp, table, ln)
    outs = [K.paged_attention_decode(q, kp, vp, table, ln) for _ in range(200)]
    assert all(torch.equal(first, x) for x in outs)
    hk, hv = (opaged.gather(host(p), host(table)[0], 32749) for p in (kp, vp))
    want, bound = oracle_rows(q, lambda b: (hk, hv), [0, 1], 128 ** -0.5, True, BF, DECODE_WEIGHT)
    check("long context", first, want, bound)


def test_empty_calls(cuda_device):
    dev = cuda_device
    z = torch.zeros(0, 4, 64, device=dev, dtype=BF)
    assert K.packed_attention(z, z, z, ints([0, 0], dev)).shape == (0, 4, 64)
    q = normal(150, 3, 4, 64, device=dev)
    out = K.packed_attention(q, z, z, ints([0, 3], dev), ints([0, 0], dev))
    assert out.shape == q.shape and bool((out == 0).all())


def test_refusals_on_the_device(cuda_device):
    dev = cuda_device
    kp, vp, table = make_cache(151, [20], 2, 64, 16, BF, dev)
    q, ln = normal(152, 1, 4, 64, device=dev), ints([20], dev)
    for bad in (dict(q=q.cpu()), dict(q=q.float()), dict(q=q[:, :3]), dict(table=table.long()), dict(ln=ln.long()),
                dict(ln=ints([1, 1], dev)), dict(kp=kp.half()), dict(q=q.repeat(2, 1, 1)), dict(vp=vp[:1]),
                dict(q=q.clone().requires_grad_()), dict(out=torch.empty(1, 4, 64, device=dev)),
                dict(status=torch.zeros(1, device=dev)), dict(q=q.expand(1, 4, 64).transpose(1, 2))):
        a = {"q": q, "kp": kp, "vp": vp, "table": table, "ln": ln, "out": None, "status": None} | bad
        with pytest.raises(ValueError):
            K.paged_attention_decode(a["q"], a["kp"], a["vp"], a["table"], a["ln"], out=a["out"], status=a["status"])
        cu = ints([0, 1], dev)
        with pytest.raises(ValueError):
            K.paged_attention_prompt(a["q"], a["kp"], a["vp"], a["table"], a["ln"], cu[:1] if a["q"].shape[0] == 2 else cu,
                                     out=a["out"], status=a["status"])
    k = normal(153, 5, 2, 64, device=dev)
    for bad in (dict(k=k[:, :, :32]), dict(v=k[:4]), dict(k=k.half(), v=k.half()), dict(cu=ints([0], dev)),
                dict(cu=torch.tensor([0, 1], device=dev)), dict(k=k[:, :1].expand(5, 2, 64))):
        a = {"k": k, "v": k, "cu": ints([0, 1], dev)} | bad
        with pytest.raises(ValueError):
            K.packed_attention(q, a["k"], a["v"], a["cu"], ints([0, 5], dev))


def test_inputs_that_require_a_gradient_are_refused(cuda_device):
    dev = cuda_device
    kp, vp, table = make_cache(154, [20], 2, 64, 16, BF, dev)
    q, ln, cu = normal(155, 1, 4, 64, device=dev), ints([20], dev), ints([0, 1], dev)
    k = normal(156, 5, 2, 64, device=dev)
    qkv, w = normal(157, 1, 8 * 64, device=dev), normal(158, 64, device=dev)
    cos, sin = (t.to(BF).to(dev) for t in rope_tables(32, 64))
    calls = [(K.paged_attention_decode, [q, kp, vp, table, ln]), (K.paged_attention_prompt, [q, kp, vp, table, ln, cu]),
             (K.packed_attention, [q, k, k, cu, ints([0, 5], dev)]),
             (K.qk_rope_paged, [qkv, w, w, cos, sin, kp, vp, table, ln, None, EPS])]
    for call, args in calls:
        for i, x in enumerate(args):
            if not isinstance(x, torch.Tensor) or x.dtype != BF or x is cos or x is sin:
                continue
            with_grad = args[:i] + [x.detach().clone().requires_grad_()] + args[i + 1:]
            with pytest.raises(ValueError, match="no backward pass"):
                call(*with_grad)
            with torch.no_grad():
                call(*with_grad)


def test_out_in_the_queries_memory_is_refused(cuda_device):
    dev = cuda_device
    kp, vp, table = make_cache(159, [20, 3], 2, 64, 16, BF, dev)
    memory = normal(160, 5, 4, 64, device=dev)
    q, ln, cu = memory[1:3], ints([20, 3], dev), ints([0, 1, 2], dev)
    k = normal(161, 5, 2, 64, device=dev)
    for out in (q, memory[:2], memory[2:4]):
        for call in (lambda o: K.paged_attention_decode(q, kp, vp, table, ln, out=o),
                     lambda o: K.paged_attention_prompt(q, kp, vp, table, ln, cu, out=o),
                     lambda o: K.packed_attention(q, k, k, cu, ints([0, 3, 5], dev), out=o)):
            with pytest.raises(ValueError, match="memory"):
                call(out)
            call(memory[3:])


def test_rows_with_a_value_that_is_not_finite_in_a_very_long_cache(cuda_device):
    """640,000 keys: rows that are computed again, one by one, take seconds, which is no expired wait. All pages
    hold the same rows (the first with one element that is not finite), so that key j of a page counts as often
    as a row sees it."""
    dev, nq, nkv, d, page, n, long = cuda_device, 4, 1, 128, 64, 64, 10000
    kp, vp = normal(162, 2, nkv, page, d, device=dev), normal(163, 2, nkv, page, d, device=dev)
    kp[1], vp[1] = kp[0], vp[0]
    vp[1, 0, 5, 3] = float("nan")
    batch = 80  # enough items that none is cut
    table = torch.zeros(batch, long, device=dev, dtype=torch.int32)
    table[0, 0] = 1
    lens, new = [long * page] + [page] * (batch - 1), [n] + [1] * (batch - 1)
    q = normal(164, sum(new), nq, d, device=dev)
    native.error_word(clear=True)
    got = K.paged_attention_prompt(q, kp, vp, table, ints(lens, dev), offsets(new, dev))
    assert native.error_word() == 0
    assert torch.isnan(got[:n, :, 3]).all()
    got[:n, :, 3] = 0
    hk, hv = (host(x[0]).transpose(1, 0, 2) for x in (kp, vp))
    want, bound = oracle_rows(q, lambda b: (hk, hv), [0] + list(range(n, n + batch)), d ** -0.5, False, BF, UNIT[BF])
    for t in range(n):
        seen = long * page - n + t + 1
        p = np.exp(d ** -0.5 * host(q)[t] @ hk[:, 0].T) * (seen // page + (np.arange(page) < seen % page))
        p /= p.sum(-1, keepdims=True)
        want[t] = p @ hv[:, 0]
        # a rounding of the weights' sum and one of an element's for every key that is added
        bound[t] = UNIT[BF] * np.abs(want[t]) + 2 * 2.0 ** -24 * seen * (p @ np.abs(hv[:, 0]))
    want[:n, :, 3] = 0
    check("very long", got, want, bound)


@pytest.mark.parametrize("tokens_each,nq", [(700, 4), (9, 2)])
def test_empty_sequences_between_others_change_nothing(cuda_device, tokens_each, nq):
    """A padded batch: blocks without an item outnumber the others, and are taken by those."""
    dev, d = cuda_device, 64
    real = [tokens_each - 3 * i for i in range(3)]
    new = [0] * 5 + [real[0]] + [0] * 1200 + [real[1], real[2]] + [0] * 3000
    q, k, v = (normal(170 + i, sum(real) + 11, nq, d, device=dev) for i in range(3))
    out = torch.full_like(q, 7.0)
    K.packed_attention(q, k, v, offsets(new, dev), out=out)
    assert bool((out[sum(real):] == 7.0).all())  # rows behind the last sequence
    cu = [0] + list(np.cumsum(real))
    hk, hv = host(k), host(v)
    want, bound = oracle_rows(q[:cu[-1]], lambda b: (hk[cu[b]:cu[b + 1]], hv[cu[b]:cu[b + 1]]), cu, d ** -0.5, True, BF, UNIT[BF])
    check("padded batch", out[:cu[-1]], want, bound)

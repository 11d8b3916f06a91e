"""The paged cache's operators on a B200 at the ends of their range: scores far apart, infinitely low ones, slots
without a sequence, outputs in the memory of inputs. Against float64, as in ``test_gpu_paged.py``."""
import numpy as np
import pytest
import torch

from paged_cases import UNIT, check, host, ints, make_cache, normal, offsets, oracle_rows

from moss_tts._runtime import kernels as K, native
from moss_tts._runtime.engine import rope_tables

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


def _first_element(dev, dtype, n, heads, d):
    q = torch.zeros(n, heads, d, device=dev, dtype=dtype)
    q[..., 0] = 1
    return q


# ------------------------------------------------------------------------------------ infinitely low scores
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,heads,keys", [(48, 16, 60), (48, 16, 128), (48, 16, 300), (48, 16, 3000), (3, 4, 60), (3, 4, 300),
                                          (3, 4, 3000)])
@pytest.mark.parametrize("others", [0.0, -120.0, 60.0])
def test_keys_of_infinitely_low_score_count_for_nothing(cuda_device, dtype, n, heads, keys, others):
    """Keys with an element of -inf against a positive one of the queries have a weight of 0, wherever they
    stand (the first key, the first of a tile, whole tiles); the others keep theirs, whose scores lie around
    ``others``. The prompt forms and the decode give what float64 gives without those keys."""
    dev, d = cuda_device, 128
    q = normal(320, n, heads, d, dtype=dtype, device=dev)
    q[..., 0] = 1
    q[..., 1] = others * d ** 0.5 / 8
    k, v = normal(321, keys, 1, d, dtype=dtype, device=dev), normal(322, keys, 1, d, dtype=dtype, device=dev)
    k[:, 0, 1] = 8
    for low in ([0], [0, 1, 2, keys - 1], list(range(0, keys, 128)), list(range(min(128, keys - 1))), list(range(0, keys, 2))):
        kk = k.clone()
        kk[low, 0, 0] = -float("inf")
        rest = np.setdiff1d(np.arange(keys), low)
        want, bound = oracle_rows(q, lambda b: (host(k)[rest], host(v)[rest]), [0, n], d ** -0.5, False, dtype, UNIT[dtype])
        got = K.packed_attention(q, kk, v, offsets([n], dev), offsets([keys], dev), causal=False)
        check(f"{len(low)} of {keys} keys infinitely low {dtype}", got, want, bound)
        pages = -(-keys // 64)
        pool = torch.zeros(2, pages * 64, 1, d, device=dev, dtype=dtype)
        pool[0, :keys], pool[1, :keys] = kk, v
        kp, vp = pool.view(2, pages, 64, 1, d).transpose(2, 3).contiguous()
        table = torch.arange(pages, device=dev, dtype=torch.int32)[None].repeat(n, 1)
        length = torch.full((n,), keys, device=dev, dtype=torch.int32)
        check("decode", K.paged_attention_decode(q, kp, vp, table, length), want, bound)
        got = K.paged_attention_prompt(q, kp, vp, table, length, offsets([1] * n, dev))
        check("prompt over pages", got, want, bound)


def test_rows_of_infinitely_low_scores_alone(cuda_device):
    """Where every key's weight is 0 the row is zeros, by either entry point, also in cut items."""
    dev, d = cuda_device, 128
    for n, keys in ((40, 100), (40, 2000), (2, 2000)):
        q = _first_element(dev, BF, n, 16, d)
        k, v = torch.zeros(keys, 1, d, device=dev, dtype=BF), normal(330, keys, 1, d, device=dev)
        k[..., 0] = -float("inf")
        got = K.packed_attention(q, k, v, offsets([n], dev), offsets([keys], dev), causal=False)
        assert bool((got == 0).all())


# ------------------------------------------------------------------------------------ scores far apart
def _raised(dev, dtype, d, keys, raised):
    """Keys whose first element is 0 but for ``raised`` {index: element}, values of 0.25 but 1.5 at those."""
    k = torch.zeros(keys, 1, d, device=dev, dtype=dtype)
    v = torch.full((keys, 1, d), 0.25, device=dev, dtype=dtype)
    for at, x in raised.items():
        k[at, 0, 0], v[at] = x, 1.5
    return k, v


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,heads,d", [(40, 16, 64), (6, 4, 128), (24, 32, 128)])  # over 512 rows, and fewer
@pytest.mark.parametrize("rise", [30.0, 60.0, 87.3, 87.4, 88.0, 88.7, 95.0, 300.0])
def test_one_key_far_above_the_others(cuda_device, dtype, n, heads, d, rise):
    """One weight of e^rise beside some of 1, in the first key tile, a later one, the last one; with the first
    key, whose score the reference may start from, among the low ones."""
    dev = cuda_device
    q = _first_element(dev, dtype, n, heads, d)
    for keys, at in ((200, 50), (200, 100), (300, 150), (300, 299), (1000, 70), (1000, 700), (3000, 2999), (100, 99)):
        k, v = _raised(dev, dtype, d, keys, {at: 1.0})
        got = K.packed_attention(q, k, v, offsets([n], dev), offsets([keys], dev), causal=False, scale=rise)
        want, bound = oracle_rows(q, lambda b: (host(k), host(v)), [0, n], rise, False, dtype, UNIT[dtype])
        check(f"rise of {rise} at {at} of {keys} {dtype}", got, want, bound)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n,heads", [(20, 4), (48, 16)])
@pytest.mark.parametrize("rise", [30.0, 88.0, 88.7, 200.0])
def test_raised_keys_of_cut_items_are_weighed_against_one_another(cuda_device, dtype, n, heads, rise):
    """Pieces of an item start from references far apart, with their largest weights anywhere."""
    dev, d, keys = cuda_device, 128, 3000
    q = _first_element(dev, dtype, n, heads, d)
    r = np.random.default_rng(310)
    cases = [{0: 1.0, 2990: 0.9921875}, {2990: 0.9921875, 400: 1.0, 384: 1.0}, {768: 1.0, 100: 0.9921875}]
    cases += [{int(at): float(x) for at, x in zip(r.integers(0, keys, 6), r.choice([1.0, 0.9921875, 0.984375, -1.0], 6))}
              for _ in range(8)]
    for raised in cases:
        k, v = _raised(dev, dtype, d, keys, raised)
        v += 0.125 * torch.arange(keys, device=dev)[:, None, None].remainder(7).to(dtype)
        got = K.packed_attention(q, k, v, offsets([n], dev), offsets([keys], dev), causal=False, scale=rise)
        want, bound = oracle_rows(q, lambda b: (host(k), host(v)), [0, n], rise, False, dtype, UNIT[dtype])
        check(f"pieces, rise of {rise} at {raised} {dtype}", got, want, bound)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rise", [20.0, 100.0])
@pytest.mark.parametrize("batch", [1, 40])  # cut along the keys, and not
def test_scores_far_above_the_first_cost_no_more_than_others(cuda_device, dtype, rise, batch):
    """Finite scores, however far apart, are no reason to compute rows again one by one: that would take a
    thousand times as long as the call, where four times is allowed here."""
    dev, d, n, heads, keys = cuda_device, 128, 40, 16, 2000
    q = _first_element(dev, dtype, n * batch, heads, d)
    cu, cu_k = offsets([n] * batch, dev), offsets([keys] * batch, dev)
    v = normal(311, keys * batch, 1, d, dtype=dtype, device=dev)

    def time_of(at):
        k = torch.zeros(keys, 1, d, device=dev, dtype=dtype)
        k[at:, 0, 0] = torch.arange(keys - at, device=dev).remainder(2).to(dtype)
        k = k.repeat(batch, 1, 1)
        best = float("inf")
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            K.packed_attention(q, k, v, cu, cu_k, causal=False, scale=rise)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    level = time_of(keys)  # no key is raised
    for at in (1, 60, 100, 130, 500, 1990):
        assert time_of(at) <= 4 * level + 0.05, (at, level)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("batch,longest", [(5, 2000), (400, 150)])
def test_items_with_scores_far_apart_among_others(cuda_device, dtype, causal, batch, longest):
    """Some sequences have keys far above their others, most have none: each gets what float64 gives it, and the
    same bits from every call."""
    dev, d, heads, rise = cuda_device, 64, 8, 100.0
    r = np.random.default_rng(312)
    new = [int(x) for x in r.integers(1, longest // 3, batch)]
    lens = [n + int(x) for n, x in zip(new, r.integers(0, longest // 2, batch))]
    q = _first_element(dev, dtype, sum(new), heads, d)
    k = torch.zeros(sum(lens), 2, d, dtype=dtype)
    at = np.concatenate(([0], np.cumsum(lens)))
    for b in range(batch):
        if b % 3 == 1:
            for i in r.integers(0, lens[b], 3):
                k[at[b] + i, int(r.integers(2)), 0] = float(r.choice([1.0, 0.9921875, 0.5, -1.0]))
    k, v = k.to(dev), normal(313, sum(lens), 2, d, dtype=dtype, device=dev)
    cu, cu_k = offsets(new, dev), offsets(lens, dev)
    got = K.packed_attention(q, k, v, cu, cu_k, causal=causal, scale=rise)
    for _ in range(5):
        assert torch.equal(got, K.packed_attention(q, k, v, cu, cu_k, causal=causal, scale=rise))
    hk, hv = host(k), host(v)
    want, bound = oracle_rows(q, lambda b: (hk[at[b]:at[b + 1]], hv[at[b]:at[b + 1]]), np.concatenate(([0], np.cumsum(new))),
                              rise, causal, dtype, UNIT[dtype])
    check(f"far apart among others {dtype} causal {causal}", got, want, bound)


# ------------------------------------------------------------------------------------ slots without a sequence
@pytest.mark.parametrize("dtype,nq,nkv,d,page", [(BF, 32, 8, 128, 64), (HF, 3, 1, 64, 16), (BF, 7, 1, 64, 256)])
@pytest.mark.parametrize("lens", [[0, 40], [0], [5, 0, 0, 33, 0]])
def test_a_step_with_empty_slots(cuda_device, dtype, nq, nkv, d, page, lens):
    """A padded decode step: a slot of length 0 is no error to the write, its query row is zeros whatever its
    q | k | v holds, no page changes for it, and the attention gives zeros; the others are as without it."""
    dev = cuda_device
    live = [b for b, n in enumerate(lens) if n]
    kp, vp, table = make_cache(340, lens, nkv, d, page, dtype, dev)
    qkv = normal(341, len(lens), (nq + 2 * nkv) * d, dtype=dtype, device=dev)
    qkv[[b for b, n in enumerate(lens) if not n]] = float("nan")
    w = torch.ones(d, device=dev, dtype=dtype)
    cos, sin = (t.to(dev) for t in rope_tables(64, d))
    cos, sin = cos.to(dtype), sin.to(dtype)
    alone = kp.clone(), vp.clone()
    ln, status = ints(lens, dev), ints([0], dev)
    out = torch.full((len(lens), nq, d), 7.0, device=dev, dtype=dtype)
    q = K.qk_rope_paged(qkv, w, w, cos, sin, kp, vp, table, ln, None, 1e-6, out=out, status=status)
    assert int(status.item()) == 0
    assert all(bool((q[b] == 0).all()) for b in range(len(lens)) if b not in live)
    if live:
        want = K.qk_rope_paged(qkv[live], w, w, cos, sin, *alone, table[live], ln[live], None, 1e-6)
        assert torch.equal(q[live], want)
    assert torch.equal(kp.nan_to_num(9.0), alone[0].nan_to_num(9.0))
    assert torch.equal(vp.nan_to_num(9.0), alone[1].nan_to_num(9.0))
    got = K.paged_attention_decode(q, kp, vp, table, ln, status=status)
    assert int(status.item()) == 0 and bool(torch.isfinite(got).all())
    assert all(bool((got[b] == 0).all()) for b in range(len(lens)) if b not in live)


def test_a_position_outside_the_tables_is_still_said(cuda_device):
    """What is an error beside an empty slot: a length beyond the tables, a negative one, and a token that
    offsets give to a sequence of length 0."""
    dev, nq, nkv, d = cuda_device, 4, 2, 128
    kp, vp, table = make_cache(342, [40, 40], nkv, d, 16, BF, dev, rubbish=0.5)
    qkv, w = normal(343, 2, (nq + 2 * nkv) * d, device=dev), torch.ones(d, device=dev, dtype=BF)
    cos, sin = (t.to(dev).to(BF) for t in rope_tables(64, d))
    before = kp.clone(), vp.clone()
    for lens, cu in (([49, 0], None), ([0, 49], None), ([0, -1], None), ([0, 0], offsets([1, 1], dev))):
        status = ints([0], dev)
        K.qk_rope_paged(qkv, w, w, cos, sin, kp, vp, table, ints(lens, dev), cu, 1e-6, status=status)
        assert int(status.item()) == 1
        assert torch.equal(kp, before[0]) and torch.equal(vp, before[1])


# ------------------------------------------------------------------------------------ memory of inputs
def test_outputs_in_the_memory_of_keys_values_and_pages_are_refused(cuda_device):
    dev, nq, nkv, d, page = cuda_device, 4, 2, 64, 16
    pool = normal(350, 2, 8, nkv, page, d, device=dev)  # keys and values
    kp, vp = pool[0], pool[1]
    table, ln, cu = ints([[0, 1], [2, 3]], dev), ints([20, 3], dev), offsets([1, 1], dev)
    q = normal(351, 2, nq, d, device=dev)
    qkv, w = normal(352, 2, (nq + 2 * nkv) * d, device=dev), torch.ones(d, device=dev, dtype=BF)
    cos, sin = (t.to(dev).to(BF) for t in rope_tables(32, d))
    before = pool.clone()
    flat = pool.view(-1)
    for first in (0, 4096, pool[0].numel() + 64):
        out = flat[first:first + q.numel()].view(q.shape)
        for call in (lambda: K.paged_attention_decode(q, kp, vp, table, ln, out=out),
                     lambda: K.paged_attention_prompt(q, kp, vp, table, ln, cu, out=out),
                     lambda: K.qk_rope_paged(qkv, w, w, cos, sin, kp, vp, table, ln, None, 1e-6, out=out)):
            with pytest.raises(ValueError, match="memory"):
                call()
    rows = normal(353, 12, nq + 2 * nkv, d, device=dev)
    k, v = rows[4:, nq:nq + nkv], rows[4:, nq + nkv:]
    cu_k = ints([0, 3, 5], dev)
    for first, ends in ((4, True), (10, True), (0, False)):  # whole rows, k and v among them
        out = rows.view(-1)[first * rows.stride(0):][:q.numel()].view(q.shape)
        if ends:
            with pytest.raises(ValueError, match="memory"):
                K.packed_attention(q, k, v, cu, cu_k, out=out)
        else:
            K.packed_attention(q, k, v, cu, cu_k, out=out)
    inside = flat[:qkv.numel()].view(qkv.shape)
    with pytest.raises(ValueError, match="memory"):
        K.qk_rope_paged(inside, w, w, cos, sin, kp, vp, table, ln, None, 1e-6)
    assert torch.equal(pool, before)


def test_second_passes_in_a_graph_and_on_two_streams(cuda_device):
    """Items that go round again, captured once and replayed on two streams at once, whole and cut: the bits of
    the plain calls, and no wait expires."""
    dev, d, heads, rise = cuda_device, 128, 8, 120.0
    native.error_word(clear=True)
    sides = []
    for side, (new, lens) in enumerate((([60, 1, 300], [900, 700, 300]), ([40], [3000]))):
        q = normal(360 + side, sum(new), heads, d, device=dev) * 0.01
        q[..., 0] = 1
        k, v = normal(362 + side, sum(lens), 1, d, device=dev) * 0.01, normal(364 + side, sum(lens), 1, d, device=dev)
        k[..., 0] = 0
        k[5::97, :, 0] = 1
        cu, cu_k = offsets(new, dev), offsets(lens, dev)
        plain = K.packed_attention(q, k, v, cu, cu_k, scale=rise)
        out, stream, graph = torch.zeros_like(q), torch.cuda.Stream(dev), torch.cuda.CUDAGraph()
        torch.cuda.synchronize(dev)
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(3):
                K.packed_attention(q, k, v, cu, cu_k, scale=rise, out=out)
        sides.append((plain, out, stream, graph, (q, k, v, cu, cu_k)))
    for _ in range(20):
        for _, out, stream, graph, _ in sides:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
    torch.cuda.synchronize(dev)
    assert native.error_word() == 0
    for plain, out, *_ in sides:
        assert bool(torch.isfinite(plain).all()) and torch.equal(plain, out)

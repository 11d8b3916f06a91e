"""Inputs of the paged cache's tests: seeded tensors, page tables in a shuffled order, and the
comparison with the float64 oracle within its bound."""
import numpy as np
import torch

from oracle import paged as opaged

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def normal(seed, *shape, dtype=torch.bfloat16, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(device)


def host(t):
    return t.detach().double().cpu().numpy()


def offsets(lens, device="cpu"):
    return torch.tensor(np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32, device=device)


def ints(values, device="cpu"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def make_cache(seed, lens, nkv, d, page, dtype, device, spare=2, order="heads", rubbish=float("nan")):
    """(k_pages, v_pages, table) for sequences of ``lens`` tokens: normal rows where a sequence has them,
    ``rubbish`` in every other row, and page ids outside the cache behind the entries in use. ``order``
    "rows" lays the heads of a row side by side ([pages, page, heads, D], seen transposed)."""
    need = [-(-n // page) for n in lens]
    count = sum(need) + spare
    perm = np.random.default_rng(seed).permutation(count)
    table = np.full((len(lens), max(max(need), 1)), 1 << 30, dtype=np.int32)
    pools = []
    for which in range(2):
        pool = torch.full((count, nkv, page, d), rubbish, dtype=dtype)
        at = 0
        for b, n in enumerate(need):
            ids = perm[at:at + n]
            table[b, :n] = ids
            rows = normal(seed * 100 + 10 * b + which + 1, n * page, nkv, d, dtype=dtype)
            rows[lens[b]:] = rubbish
            for i, pid in enumerate(ids):
                pool[pid] = rows[i * page:(i + 1) * page].transpose(0, 1)
            at += n
        pool = pool.to(device)
        if order == "rows":
            pool = pool.transpose(1, 2).contiguous().transpose(1, 2)
        pools.append(pool)
    return pools[0], pools[1], torch.from_numpy(table).to(device)


def check(label, got, want, bound):
    """``got`` within ``bound`` of ``want`` everywhere; says how much of the bound was used."""
    got = host(got).reshape(want.shape)
    err = np.abs(got - want)
    used = float(np.max(err / np.where(bound > 0, bound, 1.0), initial=0.0, where=bound > 0))
    print(f"{label}: {used:.3f} of the bound, largest error {err.max(initial=0.0):.3g}")
    assert np.all(np.isfinite(got)), f"{label}: not finite"
    assert np.all(err <= bound), f"{label}: {used:.3f} of the bound at {np.unravel_index(np.argmax(err - bound), err.shape)}"


def oracle_rows(q, gathered, cu, scale, causal, dtype, weight_unit):
    """(out, bound) of packed queries; ``gathered(b)`` gives sequence b's keys and values in float64."""
    q = host(q)
    out, bound = np.zeros_like(q), np.zeros_like(q)
    for b in range(len(cu) - 1):
        k, v = gathered(b)
        out[cu[b]:cu[b + 1]], bound[cu[b]:cu[b + 1]] = opaged.attention(q[cu[b]:cu[b + 1]], k, v, scale, causal,
                                                                        UNIT[dtype], weight_unit)
    return out, bound

"""More of the paged-pool operators against 64 bits: workspaces of larger batches, infinities, values of rows
that others do not see, and prefixes long enough that every ring of the tensor-core kernel goes round."""
import math

import pytest
from test_gpu_paged import KINDS, Batch, T  # noqa: F401 (T is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("large,small", [((129, 8192), (128, 8192)), ((64, 2432), (64, 2304)),
                                         ((65, 2432), (64, 2304))])
def test_a_larger_batchs_workspace(T, q3lib, large, small):  # noqa: F811
    """A workspace sized for more rows or a longer prefix serves fewer, and nothing behind it changes."""
    b = Batch(T, q3lib, "e4m3", "bf16", 8, 2, 128, [1 + i % 5 for i in range(small[0])], [1] * small[0],
              prefix=small[1], seed=51, spare_rows=0)
    size = q3lib.paged_attn_workspace_size(b.pool.handle, 16, large[0], large[0], 1, large[1])
    b.ws = T.full((size + (16 << 20),), 0xFF, dtype=T.uint8, device="cuda")
    b.call()
    b.check()
    assert bool((b.ws[size:] == 0xFF).all())


def _set_value(pool, slot, d, x):
    """Value d of every KV head of a bf16 pool's V row, or the code byte of an e4m3 one's."""
    pool.v[slot // 16, :, slot % 16, d] = x


@pytest.mark.parametrize("h,group,d", [(2, 2, 128), (3, 5, 64), (1, 16, 128)])
@pytest.mark.parametrize("own,width,prefix,at", [
    ([40, 33], None, 0, "last"), ([40, 33], None, 0, "first"),        # a block a strip
    ([1300, 700], 90, 0, "last"), ([1300, 700], 90, 0, "first"),      # the line, cut among blocks
    ([40, 33], None, 300, "prefix"),                                  # a prefix in the strips
    ([40, 33], 100, 300, "prefix"), ([3, 700], 100, 2000, "prefix"),  # on the tensor cores, one row tile
])
def test_infinite_values_of_a_bf16_pool(T, q3lib, h, group, d, own, width, prefix, at):  # noqa: F811
    """+infinity and -infinity among a token's values are the results of the rows that see it, in those places
    alone; whatever the weights' low halves are. (Scores are small, so that no weight underflows.)"""
    b = Batch(T, q3lib, "bf16", "bf16", h, group, d, own, [3, 2], prefix=prefix, seed=61, q_scale=0.25)
    if width:
        b.widen(width)
    # "last": of the first sequence's newest token, seen by its last row alone.
    slot = int({"last": b.slots[0][-1], "first": b.slots[0][0],
                "prefix": b.prefix_slots[-20] if prefix else -1}[at])
    sees = {"last": [2], "first": [0, 1, 2], "prefix": [0, 1, 2, 3, 4]}[at]
    for place in (5, 40):
        _set_value(b.pool, slot, place, 0.0)
    val, err = b.want()
    _set_value(b.pool, slot, 5, math.inf)
    _set_value(b.pool, slot, 40, -math.inf)
    b.call()
    T.cuda.synchronize()
    got = b.out_buf[:5].double().view(5, h * group, d)
    want = val[:5].clone()
    want[sees, :, 5], want[sees, :, 40] = math.inf, -math.inf
    there = want.isfinite()
    assert bool((got[~there] == want[~there]).all())
    assert bool((got - want)[there].abs().le(err[:5][there]).all())


def test_infinite_values_of_many_rows(T, q3lib):  # noqa: F811
    """The same over a prefix for the rows of several tiles."""
    b = Batch(T, q3lib, "bf16", "bf16", 2, 4, 128, [5 + i % 40 for i in range(90)], [1] * 90, prefix=2500, seed=62,
              q_scale=0.25)
    slot = int(b.prefix_slots[777])
    _set_value(b.pool, slot, 5, 0.0)
    val, err = b.want()
    _set_value(b.pool, slot, 5, math.inf)
    b.call()
    T.cuda.synchronize()
    got = b.out_buf[:90].double().view(90, 8, 128)
    assert bool((got[:, :, 5] == math.inf).all())
    rest = [i for i in range(128) if i != 5]
    assert bool((got - val[:90]).abs().le(err[:90])[:, :, rest].all())


@pytest.mark.parametrize("own,width,prefix", [([40, 33], None, 0), ([1300, 700], 90, 0), ([40, 33], None, 300),
                                              ([40, 33], 100, 300)])
def test_byte_zero_is_a_power_of_two(T, q3lib, own, width, prefix):  # noqa: F811
    """A row of byte 0 has the values code * 2^-127, also for queries that make scores of it: all queries are
    +-2^115, one key has the code 448 with their signs (score 448 * 128 * 2^-12 / sqrt(128) = 1.24), the others
    are zeros (byte 0 too)."""
    b = Batch(T, q3lib, "e4m3", "bf16", 1, 1, 128, own, [1, 1], prefix=prefix, seed=63, spare_rows=0)
    if width:
        b.widen(width)
    b.q_buf.copy_(T.where(b.q_buf > 0, 2.0 ** 115, -2.0 ** 115))
    b.q_buf[1] = b.q_buf[0]
    for s in b.slots + [b.prefix_slots]:
        if len(s):
            v = b.pool.get("v", s)
            b.pool.put(s, T.zeros_like(v), v)
    slot = b.prefix_slots[7:8] if prefix else b.slots[0][7:8]
    v = b.pool.get("v", slot) + 300.0
    b.pool.put(slot, (448 * 2.0 ** -127 * b.q_buf[0].double().sign()).view(1, 1, 128), v)
    assert int(b.pool.exps[int(slot) // 16, 0, int(slot) % 16, 0]) == 0
    b.call()
    b.check()


def want_by_weight(b):
    """Batch.want with a bound that goes by what has weight in a row: fp16's smallest step cuts off at most
    2^-25 of a weighted V row's power of two where the largest of the row's is at least 2^7 times that power
    (2^-32, and a V row's codes are below twice its largest value over its power), of each key; the other terms
    are Batch.want's."""
    T, d = b.T, b.d
    val = T.zeros(b.n_q, b.h * b.group, d, dtype=T.float64, device="cuda")
    err = T.zeros_like(val)
    half = T.finfo(b.dt).eps / 2
    for s, n in enumerate(b.lens):
        slots = T.cat([b.prefix_slots, b.slots[s]])
        k, v = b.pool.get("k", slots), b.pool.get("v", slots)
        for i in range(b.counts[s]):
            most = b.prefix + max(0, n - b.counts[s] + i + 1)
            if not most:
                continue
            r = b.starts[s] + i
            q = b.q_buf[r, :b.h * b.group * d].double().view(b.h, b.group, d)
            kk, vv = k[:most], v[:most]
            t = T.einsum("hgd,khd->hgk", q, kk) / math.sqrt(d)
            mag = T.einsum("hgd,khd->hgk", q.abs(), kk.abs()).amax(-1) / math.sqrt(d)
            p = T.softmax(t, -1)
            o, a = T.einsum("hgk,khd->hgd", p, vv), T.einsum("hgk,khd->hgd", p, vv.abs())
            rel = 2.0 ** -11 + 2.0 ** -20 + 2 * (d + 8) * 2.0 ** -24 * mag + 2 * most * 2.0 ** -24
            low = 2.0 ** -31 * most * (p * vv.abs().amax(-1).T[:, None]).amax(-1)
            val[r] = o.reshape(-1, d)
            err[r] = (half * o.abs() + (1 + half) * (rel[..., None] * a + low[..., None])).reshape(-1, d)
    return val, err


OWN_PATHS = [([40, 33], [4, 3], None, 0), ([1300, 700], [4, 1], 90, 0), ([40, 33], [8, 8], 90, 0),
             ([40, 33], [4, 3], None, 300)]


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("own,counts,width,prefix", OWN_PATHS)
@pytest.mark.parametrize("h,group,d", [(2, 2, 128), (3, 5, 64)])
def test_a_later_drafts_large_values(T, q3lib, typ, own, counts, width, prefix, h, group, d):  # noqa: F811
    """The newest token's values are 2^36 times the others': the rows before it are as without it."""
    b = Batch(T, q3lib, "e4m3", typ, h, group, d, own, counts, prefix=prefix, seed=71)
    if width:
        b.widen(width)
    val, err = want_by_weight(b)
    slot = b.slots[0][-1:]
    b.pool.put(slot, b.pool.get("k", slot), b.pool.get("v", slot) * 2.0 ** 36)
    b.call()
    T.cuda.synchronize()
    rows = [r for r in range(b.starts[-1]) if r != counts[0] - 1]
    got = b.out_buf[:, :h * group * d].double().view(-1, h * group, d)
    assert bool((got[rows] - val[rows]).abs().le(err[rows] + 2.0 ** -24 * T.finfo(b.dt).tiny).all())


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("own,counts,width,prefix", OWN_PATHS)
@pytest.mark.parametrize("h,group,d", [(2, 2, 128), (3, 5, 64)])
@pytest.mark.parametrize("where", [0, 5])
def test_large_values_without_weight(T, q3lib, typ, own, counts, width, prefix, h, group, d, where):  # noqa: F811
    """A key whose scores are far below the others' has values of 2^34: the rest is as exact as without it."""
    b = Batch(T, q3lib, "e4m3", typ, h, group, d, own, counts, prefix=prefix, seed=72)
    if width:
        b.widen(width)
    b.q_buf.abs_()
    slot = (b.prefix_slots if prefix else b.slots[0])[where:where + 1]
    # sum |q| / sqrt(d) is about 1.6 sqrt(d): scores of about -50 or less.
    b.pool.put(slot, T.full((1, h, d), -4.0, dtype=T.float64, device="cuda"), b.pool.get("v", slot) * 2.0 ** 34)
    val, err = want_by_weight(b)
    b.call()
    T.cuda.synchronize()
    n = b.starts[-1]
    got = b.out_buf[:n, :h * group * d].double().view(n, h * group, d)
    assert bool((got - val[:n]).abs().le(err[:n] + 2.0 ** -24 * T.finfo(b.dt).tiny).all())


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("seqs", [3, 150])
def test_rows_far_below_the_prefixs_largest(T, q3lib, typ, seqs):  # noqa: F811
    """One shared token, whose scores give it no weight, has K and V rows 2^22 times the smallest of the others:
    the results are those of the others alone, within the bound of their own values. Each row's weight lies on
    one token nearly alone, so that its values come out one by one."""
    b = Batch(T, q3lib, "e4m3", typ, 2, 2, 128, [i % 3 for i in range(seqs)], [1] * seqs, prefix=900, seed=73,
              spare_rows=0).widen(100)
    b.q_buf.abs_()
    k, v = b.pool.get("k", b.prefix_slots), b.pool.get("v", b.prefix_slots)
    k[100:] = -k[100:].abs()
    k[:100] /= 16.0
    k[37] = 2.0
    v[37] /= 16.0 * v[37].abs().amax(-1, keepdim=True)  # the smallest row
    b.pool.put(b.prefix_slots, k, v)
    slot = b.prefix_slots[100:101]  # of the same tile
    page, off = b.prefix_slots // 16, b.prefix_slots % 16
    least = b.pool.exps[page, :, off].amin(0).double() - 127  # [heads, K and V]
    b.pool.put(slot, *((sign * 448.0 * T.exp2(least[:, i] + 22)).view(1, 2, 1).expand(1, 2, 128)
                       for i, sign in enumerate((-1.0, 1.0))))
    val, err = b.want(gone=slot.tolist())
    b.call()
    T.cuda.synchronize()
    got = b.out_buf.double().view(-1, 4, 128)
    assert bool((got - val).abs().le(err + 2.0 ** -24 * T.finfo(b.dt).tiny).all())


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("seqs,d,prefix", [(5, 128, 2900), (5, 64, 4500), (140, 128, 2700), (140, 64, 2900)])
def test_many_tiles_a_block(T, q3lib, kind, typ, seqs, d, prefix):  # noqa: F811
    """148 KV heads leave a block each, and every block 21 to 36 tiles of 128 keys, odd numbers among them: one
    row tile in two streams, and pairs of row tiles. Scores grow along the prefix, so that the maxima move
    all the way, and some pages are not there."""
    b = Batch(T, q3lib, kind, typ, 148, 1, d, [(3 * i) % 20 for i in range(seqs)], [1] * seqs, prefix=prefix,
              seed=81, spare_rows=0, q_scale=1.0).widen(100)
    k = b.pool.get("k", b.prefix_slots)
    b.pool.put(b.prefix_slots, k * T.linspace(0.1, 3.0, prefix, device="cuda", dtype=T.float64)[:, None, None],
               b.pool.get("v", b.prefix_slots))
    for page in (20, 99):
        b.prefix_table[page] = -1 - page
    gone = T.cat([b.prefix_slots[16 * page:16 * page + 16] for page in (20, 99)])
    b.call()
    b.check(gone=gone.tolist())


@pytest.mark.parametrize("own,width,prefix", [([40, 33], None, 0), ([1300, 700], 90, 0), ([40, 33], None, 300),
                                              ([40, 33], 100, 300)])
@pytest.mark.parametrize("power", [-110, 100])
def test_tiny_and_large_queries(T, q3lib, own, width, prefix, power):  # noqa: F811
    """Queries of 2^-110 over keys of 2^110 have ordinary scores, and so have those of 2^100 over 2^-100."""
    b = Batch(T, q3lib, "e4m3", "bf16", 2, 2, 128, own, [2, 1], prefix=prefix, seed=91, q_scale=2.0 * 2.0 ** power)
    if width:
        b.widen(width)
    for s in b.slots + [b.prefix_slots]:
        if len(s):
            b.pool.put(s, b.pool.get("k", s) * 2.0 ** -power, b.pool.get("v", s))
    b.call()
    b.check()

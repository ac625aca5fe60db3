"""The paged-pool operators (q3_kv_write, q3_kv_read, q3_paged_attn, q3_prefix_attn,
q3_verify_drafts) against plain computations in 64 bits, through the C ABI."""
import math

import pytest

pytestmark = pytest.mark.gpu

PAGE = 16


@pytest.fixture(scope="module")
def T():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch


def _gen(T, seed):
    g = T.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _type(T, q3, name):
    return {"f32": (T.float32, q3.TYPE_F32), "bf16": (T.bfloat16, q3.TYPE_BF16),
            "f16": (T.float16, q3.TYPE_F16)}[name]


# ------------------------------------------------------------------ the pool in 64 bits

def quantise(T, x):
    """Rows in 64 bits -> (values of the codes, bytes), from the definition."""
    big = T.where(T.isfinite(x), x.abs(), T.zeros_like(x)).amax(-1)
    e = T.full(big.shape, -127, device=x.device, dtype=T.int64)
    while bool((big > 448 * T.exp2(e.double())).any()):
        e += (big > 448 * T.exp2(e.double())).long()
    y = (x / T.exp2(e.double())[..., None]).clamp(-448, 448)
    step = T.exp2(T.floor(T.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return T.where(y.isnan(), y, T.round(y / step) * step), e + 127


class Pool:
    """A pool whose every unused byte is NaN (or, as bf16, infinity)."""

    def __init__(self, T, q3, kind, n_pages, h, d):
        self.T, self.kind, self.n_pages, self.h, self.d = T, kind, n_pages, h, d
        if kind == "e4m3":
            self.k = T.full((n_pages, h, PAGE, d), 0x7F, dtype=T.uint8, device="cuda")
            self.v = T.full((n_pages, h, PAGE, d), 0xFF, dtype=T.uint8, device="cuda")
            self.exps = T.full((n_pages, h, PAGE, 2), 200, dtype=T.uint8, device="cuda")
        else:
            self.k = T.full((n_pages, h, PAGE, d), math.inf, dtype=T.bfloat16, device="cuda")
            self.v = T.full((n_pages, h, PAGE, d), math.nan, dtype=T.bfloat16, device="cuda")
            self.exps = None
        self.handle = q3.KvPool(self.k.data_ptr(), self.v.data_ptr(),
                                self.exps.data_ptr() if kind == "e4m3" else None, n_pages, h, d,
                                q3.TYPE_E4M3 if kind == "e4m3" else q3.TYPE_BF16)

    def put(self, slots, k, v):
        """Rows [n, h, d] in 64 bits into the slots."""
        T = self.T
        page, off = slots // PAGE, slots % PAGE
        for i, (to, x) in enumerate(((self.k, k), (self.v, v))):
            if self.kind == "bf16":
                to[page, :, off] = x.to(T.bfloat16)
            else:
                codes, byte = quantise(T, x)
                to[page, :, off] = codes.float().to(T.float8_e4m3fn).view(T.uint8)
                self.exps[page, :, off, i] = byte.to(T.uint8)

    def get(self, which, slots):
        """[n, h, d] in 64 bits of the slots."""
        T = self.T
        page, off = slots // PAGE, slots % PAGE
        rows = (self.k if which == "k" else self.v)[page, :, off]
        if self.kind == "bf16":
            return rows.double()
        e = self.exps[page, :, off, 0 if which == "k" else 1].double() - 127
        return rows.view(T.float8_e4m3fn).double() * T.exp2(e)[..., None]


def same(T, a, b):
    """Equal values, NaN equal to NaN."""
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ------------------------------------------------------------------ write and read

@pytest.mark.parametrize("kind", ["e4m3", "bf16"])
@pytest.mark.parametrize("typ", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,h,d,pad", [(1, 8, 128, 0), (37, 3, 64, 5), (64, 1, 64, 0), (33, 5, 128, 8),
                                       (515, 8, 128, 1)])
def test_write_then_read(T, q3lib, kind, typ, n, h, d, pad):
    """Codes and bytes are the definition's; reading gives their values rounded once; other slots and
    the columns behind a row stay as they were."""
    g = _gen(T, n + d)
    dt, code = _type(T, q3lib, typ)
    pool = Pool(T, q3lib, kind, n // PAGE + 3, h, d)
    width = h * d + pad
    k, v = (T.randn(n, width, generator=g, device="cuda")
            * T.exp2(T.randint(-9, 9, (n, 1), generator=g, device="cuda")) for _ in range(2))
    k, v = k.to(dt), v.to(dt)
    k[0, :d] = 0
    slots = T.randperm(pool.n_pages * PAGE, generator=g, device="cuda")[:n].int()
    if n > 8:  # padding, and slots past the pool's end
        slots[2], slots[3], slots[n - 1] = -1, pool.n_pages * PAGE, 2 ** 31 - 1
    fine = (slots >= 0) & (slots < pool.n_pages * PAGE)
    want = Pool(T, q3lib, kind, pool.n_pages, h, d)
    want.put(slots[fine].long(), *(x[fine][:, :h * d].reshape(-1, h, d).double() for x in (k, v)))
    q3lib.kv_write(pool.handle, k.data_ptr(), v.data_ptr(), code, width, width, slots.data_ptr(), n)
    if kind == "e4m3":
        for a, b in ((pool.k, want.k), (pool.v, want.v)):
            assert same(T, a.view(T.float8_e4m3fn).float(), b.view(T.float8_e4m3fn).float())
        assert T.equal(pool.exps, want.exps)
    else:
        for a, b in ((pool.k, want.k), (pool.v, want.v)):
            assert same(T, a.float(), b.float())
    for out_typ in ("f32", "bf16", "f16"):
        dt, code = _type(T, q3lib, out_typ)
        k2, v2 = (T.full((n, width), 7, dtype=dt, device="cuda") for _ in range(2))
        q3lib.kv_read(pool.handle, k2.data_ptr(), v2.data_ptr(), code, width, width, slots.data_ptr(), n)
        for which, got in (("k", k2), ("v", v2)):
            x = want.get(which, slots.clamp(0, pool.n_pages * PAGE - 1).long())
            x = T.where(fine[:, None, None], x, T.zeros_like(x))
            assert same(T, got[:, :h * d], x.reshape(n, h * d).to(dt))
            assert bool((got[:, h * d:] == 7).all())


def test_write_borders(T, q3lib):
    """Rows whose largest value sits at a border of the byte, ties, subnormals, the largest floats,
    zeros, infinities and NaN."""
    d = 64
    f = T.finfo(T.float32)
    tops = [448.0, 448.00003, 447.9, 1.75, 1.7500001, 2.0, 1.9999999, f.max, f.tiny, f.tiny / 2 ** 20,
            2.0 ** -149, 0.0, 3e-39, 2.0 ** -118, 2.0 ** -119, math.inf, -math.inf, math.nan]
    x = T.zeros(len(tops), 1, d, device="cuda", dtype=T.float64)
    for i, t in enumerate(tops):
        base = t if math.isfinite(t) else 3.0
        x[i, 0, 0] = t
        # Halfway points of the e4m3 grid relative to the row's top, and values far below it.
        x[i, 0, 1:34] = base * (T.arange(33, device="cuda").double() + 16) / 49
        x[i, 0, 34:60] = -base * T.exp2(-T.arange(26, device="cuda").double() / 1.25)
    x = x.float()
    n = len(tops)
    pool, want = Pool(T, q3lib, "e4m3", 2, 1, d), Pool(T, q3lib, "e4m3", 2, 1, d)
    slots = T.arange(n, device="cuda", dtype=T.int32)
    want.put(slots.long(), x.double(), -x.double())
    y = -x
    q3lib.kv_write(pool.handle, x.data_ptr(), y.data_ptr(), q3lib.TYPE_F32, d, d, slots.data_ptr(), n)
    assert T.equal(pool.exps, want.exps)
    for a, b in ((pool.k, want.k), (pool.v, want.v)):
        assert same(T, a.view(T.float8_e4m3fn).float(), b.view(T.float8_e4m3fn).float())


# ------------------------------------------------------------------ attention

class Batch:
    """A ragged batch over a pool: `lens` own tokens and `counts` query rows a sequence."""

    def __init__(self, T, q3, kind, typ, h, group, d, lens, counts, prefix=0, seed=0, spare_rows=2,
                 q_scale=2.0, pad=0):
        g = _gen(T, seed)
        self.T, self.q3, self.lens, self.counts, self.prefix = T, q3, lens, counts, prefix
        self.h, self.group, self.d = h, group, d
        pages = [-(-n // PAGE) for n in lens]
        self.width = max(1, max(pages)) + 1
        pp = -(-prefix // PAGE)
        n_pages = sum(pages) + pp + 2
        self.pool = Pool(T, q3, kind, n_pages, h, d)
        ids = T.randperm(n_pages, generator=g, device="cuda")
        self.table = T.full((len(lens), self.width), 0x7FFFFFFF, dtype=T.int32, device="cuda")
        at, self.slots = 0, []
        for b, n in enumerate(lens):
            mine = ids[at:at + pages[b]]
            at += pages[b]
            self.table[b, :pages[b]] = mine.int()
            j = T.arange(n, device="cuda")
            self.slots.append(mine[j // PAGE] * PAGE + j % PAGE if n else j)
        mine = ids[at:at + pp]
        self.prefix_table = T.cat([mine.int(), T.full((1,), -5, dtype=T.int32, device="cuda")])
        j = T.arange(prefix, device="cuda")
        self.prefix_slots = mine[j // PAGE] * PAGE + j % PAGE if prefix else j
        for s in self.slots + [self.prefix_slots]:
            if len(s):
                self.pool.put(s, *(T.randn(len(s), h, d, generator=g, device="cuda", dtype=T.float64)
                                   * T.exp2(T.randint(-3, 3, (len(s), h, 1), generator=g, device="cuda"))
                                   for _ in range(2)))
        self.starts = [0]
        for c in counts:
            self.starts.append(self.starts[-1] + c)
        self.n_q, self.max_q = self.starts[-1] + spare_rows, max(1, max(counts))
        self.dt, self.code = _type(T, q3, typ)
        self.stride = h * group * d + pad
        self.q_buf = (q_scale * T.randn(self.n_q, self.stride, generator=g, device="cuda")).to(self.dt)
        self.out_buf = T.full((self.n_q, self.stride), 9, dtype=self.dt, device="cuda")
        self.q_start = T.tensor(self.starts, dtype=T.int32, device="cuda")
        self.kv_len = T.tensor(lens, dtype=T.int32, device="cuda")
        size = q3.paged_attn_workspace_size(self.pool.handle, h * group, self.n_q, len(lens), self.max_q,
                                            prefix)
        # Garbage in the workspace, and a guard behind it.
        self.ws = T.full((size + 256,), 0xFF, dtype=T.uint8, device="cuda")

    def widen(self, width):
        """The same sequences in a wider table, as one sized for longer ones."""
        T = self.T
        wide = T.full((len(self.lens), width), -9, dtype=T.int32, device="cuda")
        wide[:, :self.width] = self.table
        self.table, self.width = wide, width
        return self

    def call(self, stream=None, ws=None, out=None):
        args = [(self.out_buf if out is None else out).data_ptr(),
                (self.ws if ws is None else ws).data_ptr(), self.q_buf.data_ptr(), self.code,
                self.stride, self.stride, self.pool.handle, self.h * self.group, self.n_q,
                len(self.lens), self.max_q, self.q_start.data_ptr(), self.kv_len.data_ptr(),
                self.table.data_ptr(), self.width]
        if self.prefix:
            self.q3.prefix_attn(*args, self.prefix_table.data_ptr(), self.prefix, stream)
        else:
            self.q3.paged_attn(*args, stream)

    def want(self, gone=()):
        """(values, error bounds) [n_q, heads, d] in 64 bits; `gone`: own slots out of the attention.

        The bound: one rounding of the result to its type; the probabilities' rounding (fp16 2^-11 with
        an e4m3 pool, twice bf16's 2^-8 with a bf16 one, the two halves of a split value), exp2's 2^-21,
        the score's fp32 sum (d + 8 roundings of 2^-24 of sum |q k|, scaled, twice: numerator and
        denominator) and the fp32 sums over the keys (n of 2^-24, twice), each relative to sum p |v|;
        and half of fp16's smallest step, 2^-25, of weights whose largest is 2^8 or more, times the
        largest value that its row's byte stands for, less than twice max |v|."""
        T, d = self.T, self.d
        val = T.zeros(self.n_q, self.h * self.group, d, dtype=T.float64, device="cuda")
        err = T.zeros_like(val)
        half = T.finfo(self.dt).eps / 2
        p_half = 2.0 ** -11 if self.pool.kind == "e4m3" else 2.0 ** -16
        for b, n in enumerate(self.lens):
            s = T.cat([self.prefix_slots, self.slots[b]])
            k, v = self.pool.get("k", s), self.pool.get("v", s)
            keep = T.ones(len(s), dtype=T.bool, device="cuda")
            for x in gone:
                keep &= s != x
            for i in range(self.counts[b]):
                most = self.prefix + max(0, n - self.counts[b] + i + 1)
                there = keep[:most]
                if not bool(there.any()):
                    continue
                r = self.starts[b] + i
                q = self.q_buf[r, :self.h * self.group * d].double().view(self.h, self.group, d)
                kk, vv = k[:most][there], v[:most][there]
                t = T.einsum("hgd,khd->hgk", q, kk) / math.sqrt(d)
                mag = T.einsum("hgd,khd->hgk", q.abs(), kk.abs()).amax(-1) / math.sqrt(d)
                p = T.softmax(t, -1)
                o = T.einsum("hgk,khd->hgd", p, vv)
                a = T.einsum("hgk,khd->hgd", p, vv.abs())
                rel = (p_half + 2.0 ** -20 + 2 * (d + 8) * 2.0 ** -24 * mag + 2 * len(kk) * 2.0 ** -24)
                low = 2.0 ** -32 * len(kk) * vv.abs().amax((0, 2))[:, None, None]
                val[r] = o.reshape(-1, d)
                err[r] = (half * o.abs() + (1 + half) * (rel[..., None] * a + low)).reshape(-1, d)
        return val, err

    def check(self, gone=(), out=None):
        T, hd = self.T, self.h * self.group * self.d
        out = self.out_buf if out is None else out
        T.cuda.synchronize()
        val, err = self.want(gone)
        n = self.starts[-1]
        got = out[:n, :hd].double().view(n, -1, self.d)
        assert bool(got.isfinite().all()), "not finite"
        over = ((got - val[:n]).abs() - err[:n] - 2.0 ** -24 * T.finfo(self.dt).tiny)
        assert float(over.max()) <= 0, f"off by {float((got - val[:n]).abs().max())}, {float(over.max())} over"
        assert bool((out[n:] == 9).all()), "rows behind the last sequence"
        assert bool((out[:, hd:] == 9).all()), "columns behind a row"
        assert bool((self.ws[-256:] == 0xFF).all()), "behind the workspace"


KINDS = [("e4m3", "bf16"), ("e4m3", "f16"), ("bf16", "bf16")]
OWN = [
    ([1], [1]), ([16], [1]), ([17], [1]), ([512], [1]), ([0], [1]),
    ([5, 0, 33, 16, 1, 700], [1] * 6),
    ([5, 0, 33, 2, 1, 300], [3, 2, 3, 3, 0, 1]),  # rows before a sequence's first token, none at all
    ([2100, 31, 64], [8, 5, 8]),
]


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("h,group,d", [(8, 2, 128), (2, 5, 64), (1, 1, 128), (3, 16, 64)])
@pytest.mark.parametrize("lens,counts", OWN, ids=str)
def test_paged_attention(T, q3lib, kind, typ, h, group, d, lens, counts):
    b = Batch(T, q3lib, kind, typ, h, group, d, lens, counts, seed=len(lens) + d, pad=8)
    b.call()
    b.check()


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 127, 128, 129, 1003])
@pytest.mark.parametrize("h,group,d", [(2, 2, 128), (3, 5, 64)])
def test_prefix_attention(T, q3lib, kind, typ, prefix, h, group, d):
    b = Batch(T, q3lib, kind, typ, h, group, d, [0, 1, 40, 7, 130], [1, 1, 3, 0, 2], prefix=prefix,
              seed=prefix + d)
    b.call()
    b.check()


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("seqs,rows,h,group,prefix", [(1, 1, 8, 2, 300), (70, 1, 8, 2, 900),
                                                      (129, 2, 1, 1, 260), (40, 4, 2, 8, 2100),
                                                      (3, 2, 1, 64, 200), (150, 1, 4, 7, 640)])
def test_prefix_attention_row_tiles(T, q3lib, kind, typ, seqs, rows, h, group, prefix):
    """Rows of the batch from less than one tensor-core tile to several."""
    lens = [(7 * i) % 90 for i in range(seqs)]
    b = Batch(T, q3lib, kind, typ, h, group, 128, lens, [rows - (i % 4 == 3) for i in range(seqs)],
              prefix=prefix, seed=seqs)
    b.call()
    b.check()


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 127, 128, 129, 257, 1003])
@pytest.mark.parametrize("h,group,d", [(2, 2, 128), (3, 5, 64)])
def test_prefix_attention_behind_wide_tables(T, q3lib, kind, typ, prefix, h, group, d):
    """Tables wide enough that a short prefix too goes to the tensor cores."""
    b = Batch(T, q3lib, kind, typ, h, group, d, [0, 1, 40, 7, 130], [1, 1, 3, 0, 2], prefix=prefix,
              seed=prefix + d).widen(100)
    b.call()
    b.check()


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("seqs,rows,h,group,prefix", [(1, 1, 8, 2, 300), (129, 2, 1, 1, 260), (3, 2, 1, 64, 200),
                                                      (64, 1, 2, 2, 4099)])
def test_prefix_row_tiles_behind_wide_tables(T, q3lib, kind, typ, seqs, rows, h, group, prefix):
    lens = [(7 * i) % 90 for i in range(seqs)]
    b = Batch(T, q3lib, kind, typ, h, group, 128, lens, [rows - (i % 4 == 3) for i in range(seqs)],
              prefix=prefix, seed=seqs).widen(101)
    b.call()
    b.check()


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("wide", [False, True])
def test_prefix_of_bad_pages_alone(T, q3lib, kind, typ, wide):
    """A prefix none of whose pages is in the pool is no prefix."""
    b = Batch(T, q3lib, kind, typ, 2, 2, 128, [100, 0, 3], [2, 1, 1], prefix=200, seed=24)
    if wide:
        b.widen(99)
    b.prefix_table.fill_(b.pool.n_pages)
    b.call()
    b.check(gone=b.prefix_slots.tolist())


@pytest.mark.parametrize("kind,typ", KINDS)
def test_extremes_behind_wide_tables(T, q3lib, kind, typ):
    """Shared rows of zeros, of 2^-30 and of 2^24 beside ordinary ones, and bad pages among them."""
    b = Batch(T, q3lib, kind, typ, 2, 2, 128, [60, 200], [2, 3], prefix=300, seed=25, q_scale=1.0).widen(98)
    k, v = b.pool.get("k", b.prefix_slots), b.pool.get("v", b.prefix_slots)
    v[0] *= 2.0 ** -30
    v[1] = 0
    v[3] *= 2.0 ** (6 if typ == "f16" else 24)
    v[140] *= 2.0 ** -18
    k[5], k[6] = 0, k[6] * 2.0 ** -20
    k[0] = 4 * b.q_buf[3].double().view(2, 2, 128).mean(1)
    b.pool.put(b.prefix_slots, k, v)
    b.prefix_table[4] = -1
    b.call()
    b.check(gone=b.prefix_slots[64:80].tolist())


@pytest.mark.parametrize("kind,typ", KINDS)
def test_many_rows_and_many_short_sequences(T, q3lib, kind, typ):
    """128 rows of one KV head in a sequence, and more sequences than a block has threads."""
    b = Batch(T, q3lib, kind, typ, 2, 4, 128, [200, 500, 40], [32, 1, 17], seed=3)
    b.call()
    b.check()
    b = Batch(T, q3lib, kind, typ, 1, 2, 64, [(5 * i) % 23 for i in range(700)], [1] * 700, seed=4)
    b.call()
    b.check()


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("prefix,width", [(0, 40), (0, 90), (150, 40), (150, 110)])
def test_the_largest_group(T, q3lib, kind, typ, prefix, width):
    """64 query heads to a KV head, two rows a sequence."""
    b = Batch(T, q3lib, kind, typ, 1, 64, 128, [200, 1, 500], [2, 1, 2], prefix=prefix, seed=17).widen(width)
    b.call()
    b.check()


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("prefix", [0, 200])
def test_bad_pages_leave_the_attention(T, q3lib, kind, typ, prefix):
    b = Batch(T, q3lib, kind, typ, 2, 2, 128, [100, 33, 16], [2, 1, 1], prefix=prefix, seed=8)
    gone = [b.slots[0][32:48], b.slots[1][0:16], b.slots[2]]
    for (s, page), bad in zip(((0, 2), (1, 0), (2, 0)), (-1, b.pool.n_pages, -2 ** 31)):
        b.table[s, page] = bad
    if prefix:
        b.prefix_table[5] = 2 ** 31 - 1
        gone.append(b.prefix_slots[80:96])
    b.call()
    b.check(gone=T.cat(gone).tolist())


@pytest.mark.parametrize("kind,typ", KINDS)
def test_a_later_rows_values_do_not_reach_an_earlier_row(T, q3lib, kind, typ):
    """The cached values of a drafted token are NaN: rows before it are as without them."""
    b = Batch(T, q3lib, kind, typ, 2, 2, 128, [37, 16, 50], [4, 3, 1], prefix=0, seed=9)
    val, err = b.want()
    for s, n in ((0, 37), (1, 16)):
        slot = b.slots[s][n - 2]  # seen by the last two rows alone
        page, off = slot // PAGE, slot % PAGE
        if kind == "e4m3":
            b.pool.v[page, :, off] = 0x7F
            b.pool.k[page, :, off, 3] = 0xFF
        else:
            b.pool.v[page, :, off] = math.inf
            b.pool.k[page, :, off, 3] = math.nan
    b.call()
    T.cuda.synchronize()
    got = b.out_buf[:8, :].double().view(8, 4, 128)
    clean, dirty = [0, 1, 4, 7], [2, 3, 5, 6]
    assert bool((got[clean] - val[clean]).abs().le(err[clean]).all())
    assert bool(got[dirty].isnan().all())


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("prefix", [0, 300])
def test_extreme_magnitudes(T, q3lib, kind, typ, prefix):
    """Rows of zeros, of 2^-40 and of the largest powers beside ordinary ones; a token that takes
    nearly all of the weight and has values of 2^-30."""
    b = Batch(T, q3lib, kind, typ, 2, 2, 128, [60, 200], [2, 3], prefix=prefix, seed=10, q_scale=1.0)
    big = 2.0 ** 7 if typ == "f16" else 2.0 ** 20
    b.q_buf[0] *= 2.0 ** -14 if typ == "f16" else 2.0 ** -60
    b.q_buf[1] *= big
    b.q_buf[2] = 0
    k0 = b.pool.get("k", b.slots[0]) / big * 8  # keeps the second row's scores ordinary
    b.pool.put(b.slots[0], k0, b.pool.get("v", b.slots[0]))
    s = T.cat([b.prefix_slots, b.slots[1]])
    k, v = b.pool.get("k", s), b.pool.get("v", s)
    v[0] *= 2.0 ** -30
    v[1] = 0
    v[3] *= 2.0 ** (6 if typ == "f16" else 24)
    k[5] = 0
    k[0] = 4 * b.q_buf[3].double().view(2, 2, 128).mean(1)
    b.pool.put(s, k, v)
    if prefix:  # the first sequence's own keys shrank, its view of the prefix did not
        b.q_buf[1] /= big
    b.call()
    b.check()


@pytest.mark.parametrize("kind,typ", KINDS)
def test_offsets_past_32_bits(T, q3lib, kind, typ):
    """Pages whose byte offsets pass 2^32 (and, as bf16, whose element offsets pass 2^31)."""
    h, d, n_pages = 16, 128, 135_000  # 4.4 GB of e4m3, 8.8 GB of bf16 for K alone
    small = Batch(T, q3lib, kind, typ, h, 1, d, [40], [2], seed=11)
    pool = Pool(T, q3lib, kind, 1, h, d)
    pool.k, pool.v = (T.empty((n_pages,) + tuple(x.shape[1:]), dtype=x.dtype, device="cuda")
                      for x in (pool.k, pool.v))
    if kind == "e4m3":
        pool.exps = T.zeros((n_pages, h, PAGE, 2), dtype=T.uint8, device="cuda")
    pool.n_pages = n_pages
    pool.handle = q3lib.KvPool(pool.k.data_ptr(), pool.v.data_ptr(),
                               pool.exps.data_ptr() if kind == "e4m3" else None, n_pages, h, d,
                               pool.handle.type)
    pages = T.tensor([n_pages - 1, n_pages - 3, n_pages - 2], device="cuda")
    j = T.arange(40, device="cuda")
    slots = pages[j // PAGE] * PAGE + j % PAGE
    rows = [small.pool.get(w, small.slots[0]).float().contiguous() for w in "kv"]
    s32 = slots.int()
    q3lib.kv_write(pool.handle, rows[0].data_ptr(), rows[1].data_ptr(), q3lib.TYPE_F32, h * d, h * d,
                   s32.data_ptr(), 40)
    back = [T.empty_like(x) for x in rows]
    q3lib.kv_read(pool.handle, back[0].data_ptr(), back[1].data_ptr(), q3lib.TYPE_F32, h * d, h * d,
                  s32.data_ptr(), 40)
    assert all(T.equal(x, y) for x, y in zip(rows, back))  # values of the pool's own grid
    small.pool, small.slots = pool, [slots]
    small.table[0, :3] = pages.int()
    small.call()
    small.check()


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("prefix", [0, 150])
@pytest.mark.parametrize("width", [None, 0, 70])
def test_rows_between_sequences_and_odd_tables(T, q3lib, kind, typ, prefix, width):
    """q_start begins past 0 and leaves rows out; tables without a page, and wider than any sequence."""
    lens = [0, 0, 0] if width == 0 else [20, 33, 7]
    b = Batch(T, q3lib, kind, typ, 2, 3, 128, lens, [2, 1, 2], prefix=prefix, seed=17, spare_rows=6)
    # Rows 1, 2 | 4 | 6 of the buffer; the third sequence ends where it would run past the last row.
    b.q_start.copy_(T.tensor([1, 3, 4, 6], dtype=T.int32))
    if width == 0:
        b.width = 0
    elif width:
        b.widen(width)
    b.starts = [1, 3, 4, 6]
    b.call()
    T.cuda.synchronize()
    val, err = b.want()
    got = b.out_buf.double()[:, :6 * 128].view(-1, 6, 128)
    assert bool((got[1:6] - val[1:6]).abs().le(err[1:6] + 2.0 ** -24 * T.finfo(b.dt).tiny).all())
    assert bool((b.out_buf[0] == 9).all()) and bool((b.out_buf[6:] == 9).all())
    # A gap: the second sequence has no row, row 3 belongs to nothing.
    b.out_buf.fill_(9)
    b.q_start.copy_(T.tensor([1, 3, 3, 5], dtype=T.int32))
    b.counts, b.starts = [2, 0, 2], [1, 3, 3, 5]
    b.call()
    T.cuda.synchronize()
    val, err = b.want()
    got = b.out_buf.double()[:, :6 * 128].view(-1, 6, 128)
    assert bool((got[1:5] - val[1:5]).abs().le(err[1:5] + 2.0 ** -24 * T.finfo(b.dt).tiny).all())
    assert bool((b.out_buf[0] == 9).all()) and bool((b.out_buf[5:] == 9).all())


@pytest.mark.parametrize("kind,typ", KINDS)
def test_no_prefix_is_the_plain_call(T, q3lib, kind, typ):
    b = Batch(T, q3lib, kind, typ, 2, 2, 128, [900, 1300, 2], [3, 1, 2], seed=18)
    b.call()
    b.check()
    out = T.full_like(b.out_buf, 9)
    q3lib.prefix_attn(out.data_ptr(), b.ws.data_ptr(), b.q_buf.data_ptr(), b.code, b.stride, b.stride,
                      b.pool.handle, 4, b.n_q, 3, b.max_q, b.q_start.data_ptr(), b.kv_len.data_ptr(),
                      b.table.data_ptr(), b.width, None, 0)
    T.cuda.synchronize()
    assert T.equal(out, b.out_buf)


@pytest.mark.parametrize("kind,typ", KINDS)
@pytest.mark.parametrize("h,group,d,counts", [(4, 2, 128, [1, 1, 1]), (2, 5, 64, [2, 3, 1]), (1, 8, 128, [8, 1, 16])])
def test_long_tables_with_a_prefix(T, q3lib, kind, typ, h, group, d, counts):
    """Sequences long enough to be cut among blocks, behind a prefix."""
    b = Batch(T, q3lib, kind, typ, h, group, d, [2300, 9, 1100], counts, prefix=700, seed=19)
    b.call()
    b.check()


def test_rows_of_nan_and_infinity_stay_their_own(T, q3lib):
    """A query row that holds NaN or infinity gives NaN in its own rows and leaves the others alone."""
    for prefix in (0, 300):
        b = Batch(T, q3lib, "e4m3", "bf16", 2, 2, 128, [40, 40, 40], [1, 1, 1], prefix=prefix, seed=20)
        val, err = b.want()
        b.q_buf[0, 5] = math.nan
        b.q_buf[0, 300] = math.nan
        b.q_buf[1, ::128] = math.inf
        b.call()
        T.cuda.synchronize()
        got = b.out_buf.double()[:, :512].view(-1, 4, 128)
        assert bool(got[0, 0].isnan().all()) and bool(got[0, 2].isnan().all()) and bool(got[1].isnan().all())
        assert bool((got[0, 1::2] - val[0, 1::2]).abs().le(err[0, 1::2]).all())
        assert bool((got[2] - val[2]).abs().le(err[2]).all())


def test_a_nan_key_reaches_the_rows_that_see_it(T, q3lib):
    for kind in ("e4m3", "bf16"):
        b = Batch(T, q3lib, kind, "bf16", 2, 2, 128, [40, 40], [1, 1], prefix=300, seed=22)
        slot = b.prefix_slots[130]
        page, off = slot // PAGE, slot % PAGE
        if kind == "e4m3":
            b.pool.k[page, 1, off, 9] = 0x7F
        else:
            b.pool.k[page, 1, off, 9] = math.nan
        val, err = b.want()
        b.call()
        T.cuda.synchronize()
        got = b.out_buf.double()[:2, :512].view(2, 4, 128)
        assert bool(got[:, 2:].isnan().all())
        assert bool((got[:, :2] - val[:2, :2]).abs().le(err[:2, :2]).all())


# ------------------------------------------------------------------ streams, graphs, workspaces

@pytest.mark.parametrize("prefix,width", [(0, 60), (0, 90), (500, 60), (500, 90)])
def test_same_bits_on_any_stream_and_again(T, q3lib, prefix, width):
    b = Batch(T, q3lib, "e4m3", "bf16", 4, 2, 128, [900, 40, 333], [2, 1, 3], prefix=prefix, seed=12).widen(width)
    b.call()
    b.check()
    first = b.out_buf.clone()
    streams = [T.cuda.Stream() for _ in range(2)]
    outs = [T.full_like(first, 9) for _ in streams]
    spaces = [T.full_like(b.ws, 0x7F) for _ in streams]
    T.cuda.synchronize()
    for _ in range(3):
        for s, out, ws in zip(streams, outs, spaces):
            b.call(stream=s.cuda_stream, ws=ws, out=out)
    T.cuda.synchronize()
    assert all(T.equal(first, out) for out in outs)


@pytest.mark.parametrize("prefix,width", [(0, 30), (0, 90), (300, 30), (300, 90)])
def test_captured_step_follows_its_lengths(T, q3lib, prefix, width):
    """Two graphs over one workspace, replayed in turn, each with lengths and rows set afterwards."""
    b = Batch(T, q3lib, "e4m3", "f16", 2, 2, 128, [400, 90], [2, 2], prefix=prefix, seed=13).widen(width)
    b.call()  # as a program's eager warm-up
    T.cuda.synchronize()
    stream = T.cuda.Stream()
    graphs, outs = [], [T.full_like(b.out_buf, 9) for _ in range(2)]
    for out in outs:
        g = T.cuda.CUDAGraph()
        with T.cuda.graph(g, stream=stream):
            b.call(stream=T.cuda.current_stream().cuda_stream, out=out)
        graphs.append(g)
    for lens in ([400, 90], [3, 0], [17, 64]):
        b.lens = lens
        b.slots = [b.slots[i] if len(b.slots[i]) >= n else None for i, n in enumerate(lens)]
        full = [s.clone() for s in b.slots]
        b.slots = [s[:n] for s, n in zip(full, lens)]
        b.kv_len.copy_(T.tensor(lens, dtype=T.int32))
        for g, out in zip(graphs, outs):
            out.fill_(9)
            g.replay()
            b.check(out=out)
        b.slots = full


def test_host_pointers_are_refused(T, q3lib):
    b = Batch(T, q3lib, "e4m3", "bf16", 1, 1, 64, [5], [1], seed=14)
    host = T.zeros(64)
    with pytest.raises(q3lib.InvalidArgument, match="not device memory"):
        q3lib.kv_write(b.pool.handle, host.data_ptr(), host.data_ptr(), q3lib.TYPE_F32, 64, 64,
                       b.kv_len.data_ptr(), 1)
    host_table = T.zeros(4, dtype=T.int32)
    b.table = host_table
    with pytest.raises(q3lib.InvalidArgument, match="not device memory"):
        b.call()


# ------------------------------------------------------------------ draft verification

def verify_by_hand(target, draft, toks, counts, ua, us, vocab):
    """Token by token on the host, in 64 bits."""
    out, taken = [], []
    for b, count in enumerate(counts):
        n = 0
        while n < count:
            t = toks[b][n]
            if not 0 <= t < vocab:
                break
            q = 1.0 if draft is None else draft[b][n][t]
            if not ua[b][n] * (q if q > 0 else 0.0) < target[b][n][t]:
                break
            n += 1
        p = [x if x > 0 else 0.0 for x in target[b][n]]
        r = p
        if n < count:
            r = [max(0.0, x - (y if y > 0 else 0.0)) for x, y in
                 zip(p, draft[b][n] if draft is not None else [float(i == toks[b][n]) for i in range(vocab)])]
        if not sum(r) > 0:
            r = p
        goal, c, got = us[b] * math.fsum(r), 0.0, None
        for i, x in enumerate(r):
            c += x
            if c > goal:
                got = i
                break
        if got is None:
            got = max([i for i, x in enumerate(r) if x > 0], default=0)
        out.append(list(toks[b][:n]) + [got] + [-1] * (len(toks[b]) - n))
        taken.append(n)
    return out, taken


def run_verify(T, q3, target, draft, toks, counts, ua, us, vocab):
    b, k = toks.shape
    out = T.full((b, k + 1), -7, dtype=T.int32, device="cuda")
    acc = T.full((b,), -7, dtype=T.int32, device="cuda")
    q3.verify_drafts(out.data_ptr(), acc.data_ptr(), target.data_ptr(), target.stride(0), target.stride(1),
                     None if draft is None else draft.data_ptr(),
                     0 if draft is None else draft.stride(0), 0 if draft is None else draft.stride(1),
                     toks.data_ptr() if k else None, None if counts is None else counts.data_ptr(),
                     ua.data_ptr() if k else None, us.data_ptr(), b, k, vocab)
    T.cuda.synchronize()
    return out.tolist(), acc.tolist()


def make_verify(T, seed, b, k, vocab, pad=0, sharp=1.0):
    g = _gen(T, seed)
    logits = sharp * T.randn(b, k + 1, vocab, generator=g, device="cuda")
    target = T.empty(b, k + 1, vocab + pad, device="cuda").fill_(1e9)[:, :, :vocab]
    target.copy_(T.softmax(logits, -1))
    draft = T.empty(b, k, vocab + pad, device="cuda").fill_(1e9)[:, :, :vocab]
    draft.copy_(T.softmax(logits[:, :k] + 0.6 * T.randn(b, k, vocab, generator=g, device="cuda"), -1))
    toks = (draft / T.empty(b, k, vocab, device="cuda").exponential_(generator=g)).argmax(-1).int() if k \
        else T.zeros(b, 0, dtype=T.int32, device="cuda")
    ua, us = T.rand(b, k, generator=g, device="cuda"), T.rand(b, generator=g, device="cuda")
    counts = T.tensor([k if i % 3 else max(0, k - 1) for i in range(b)], dtype=T.int32, device="cuda")
    return target, draft, toks, counts, ua, us


@pytest.mark.parametrize("b,k,vocab,pad", [(1, 1, 1, 0), (5, 3, 2, 3), (9, 4, 1000, 0), (3, 2, 4099, 1),
                                           (2, 5, 50257, 0), (7, 0, 333, 0), (2, 8, 151936, 4),
                                           (300, 2, 64, 0)])
@pytest.mark.parametrize("certain", [False, True])
def test_verification(T, q3lib, b, k, vocab, pad, certain):
    target, draft, toks, counts, ua, us = make_verify(T, b + k, b, k, vocab, pad)
    if certain:
        draft = None
        toks = target[:, :k].argmax(-1).int() if k else toks
        ua = ua * 0.2 / max(1, vocab) ** 0.5
    got = run_verify(T, q3lib, target, draft, toks, counts, ua, us, vocab)
    want = verify_by_hand(target.double().tolist(), None if draft is None else draft.double().tolist(),
                          toks.tolist(), counts.tolist(), ua.double().tolist(), us.double().tolist(), vocab)
    assert got[1] == want[1]
    assert got[0] == [list(x) for x in want[0]]


def test_verification_edges(T, q3lib):
    """Every draft taken, none taken, tokens outside the vocabulary, empty residuals and rows, NaN, and
    the numbers 0 and 1."""
    v, k = 700, 2
    target, draft, toks, counts, ua, us = make_verify(T, 5, 12, k, v, sharp=2.0)
    counts[:] = k
    counts[3], counts[4] = -5, 99
    ua[0], ua[1] = 0.0, 0.0
    toks[2, 0], toks[3, 0], toks[5, 1] = -1, v, 2 ** 31 - 1
    draft[6] = target[6, :k]          # nothing left over: the target's own row
    toks[6, 0] = 5
    target[6, 0, 5] = 0.0
    draft[6, 0] = target[6, 0]
    draft[6, 0, 5] = 0.5
    target[7, 0] = 0.0                # nothing to draw from at all
    target[8, 0, 100:300] = math.nan
    draft[8, 0, 400:500] = math.nan
    ua[8, 0] = 1.0
    us[9], us[10], us[11] = 0.0, 1.0, 1.0 - 2.0 ** -24
    target[10, :, -50:] = 0.0
    for n_drafts in (counts, None):
        got = run_verify(T, q3lib, target, draft, toks, n_drafts, ua, us, v)
        clipped = [min(max(c, 0), k) for c in counts.tolist()] if n_drafts is not None else [k] * 12
        want = verify_by_hand(target.double().tolist(), draft.double().tolist(), toks.tolist(), clipped,
                              ua.double().tolist(), us.double().tolist(), v)
        assert got[1] == want[1]
        assert got[0] == want[0]
    assert got[0][7][0] == 0


@pytest.mark.parametrize("b,k,vocab", [(2, 40, 300), (1, 1024, 9), (20, 2, 40000)])
def test_verification_of_many_drafts(T, q3lib, b, k, vocab):
    """More drafts than a warp has lanes, all but the last few taken; more blocks than multiprocessors."""
    target, draft, toks, counts, ua, us = make_verify(T, 77, b, k, vocab)
    ua[:, :max(1, k - 3)] = 0.0
    got = run_verify(T, q3lib, target, draft, toks, counts, ua, us, vocab)
    want = verify_by_hand(target.double().tolist(), draft.double().tolist(), toks.tolist(), counts.tolist(),
                          ua.double().tolist(), us.double().tolist(), vocab)
    assert got == (want[0], want[1])
    assert min(got[1]) >= max(1, k - 3) - 1


def test_drawn_tokens_follow_the_target(T, q3lib):
    """Speculative sampling leaves the target's distribution: the first token of 40,000 sequences, each
    cell within 6 standard deviations."""
    b, v = 40_000, 8
    g = _gen(T, 21)
    p = T.softmax(T.randn(v, generator=g, device="cuda"), 0)
    q = T.softmax(T.randn(v, generator=g, device="cuda"), 0)
    target, draft = p.expand(b, 2, v).contiguous(), q.expand(b, 1, v).contiguous()
    toks = T.multinomial(q, b, replacement=True, generator=g).int()[:, None].contiguous()
    ua, us = T.rand(b, 1, generator=g, device="cuda"), T.rand(b, generator=g, device="cuda")
    out, _ = run_verify(T, q3lib, target, draft, toks, None, ua, us, v)
    n = T.bincount(T.tensor([x[0] for x in out]), minlength=v).double()
    p = p.double().cpu()
    assert bool(((n - b * p).abs() <= 6 * (b * p * (1 - p)).sqrt()).all())


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("prefix", [0, 520])
def test_a_drafting_step(T, q3lib, prefix):
    """A step of a serving loop: the rows of four drafts and the token before them go into the cache,
    attend over it, give probabilities, and are verified; then the next step goes on from what was
    accepted, its rows written over the rejected ones."""
    h, group, d, v = 2, 2, 64, 257
    b = Batch(T, q3lib, "e4m3", "bf16", h, group, d, [64, 30, 16], [5, 5, 5], prefix=prefix, seed=31,
              spare_rows=0)
    g = _gen(T, 32)
    lens = [37, 20, 5]
    proj = T.randn(h * group * d, v, generator=g, device="cuda") * 0.5
    full = [s.clone() for s in b.slots]
    for step in range(2):
        k, v_rows = (T.randn(15, h, d, generator=g, device="cuda") for _ in range(2))
        slots = T.cat([full[i][lens[i]:lens[i] + 5] for i in range(3)]).int()
        q3lib.kv_write(b.pool.handle, k.data_ptr(), v_rows.data_ptr(), q3lib.TYPE_F32, h * d, h * d,
                       slots.data_ptr(), 15)
        codes, byte = quantise(T, k.double())
        assert same(T, b.pool.get("k", slots.long()), codes * T.exp2(byte.double() - 127)[..., None])
        b.lens = [n + 5 for n in lens]
        b.slots = [s[:n] for s, n in zip(full, b.lens)]
        b.kv_len.copy_(T.tensor(b.lens, dtype=T.int32))
        b.q_buf.copy_(T.randn(b.q_buf.shape, generator=g, device="cuda"))
        b.call()
        b.check()
        target = T.softmax(b.out_buf.float() @ proj, -1).view(3, 5, v).contiguous()
        draft = T.softmax(target[:, :4].log() + T.randn(3, 4, v, generator=g, device="cuda"), -1)
        toks = draft.argmax(-1).int()
        ua, us = T.rand(3, 4, generator=g, device="cuda"), T.rand(3, generator=g, device="cuda")
        got = run_verify(T, q3lib, target, draft, toks, None, ua, us, v)
        want = verify_by_hand(target.double().tolist(), draft.double().tolist(), toks.tolist(), [4] * 3,
                              ua.double().tolist(), us.double().tolist(), v)
        assert got == (want[0], want[1])
        lens = [n + 1 + a for n, a in zip(lens, got[1])]


def test_all_at_once(T, q3lib):
    """Every operator on a stream of its own, several rounds on their way together, and once more replayed
    from one graph that forks to those streams: what each gave alone, to the bit."""
    own = Batch(T, q3lib, "e4m3", "bf16", 4, 2, 128, [900, 40, 333], [2, 1, 3], seed=41).widen(90)
    far = Batch(T, q3lib, "bf16", "bf16", 2, 4, 64, [50, 0, 9], [2, 1, 3], prefix=2000, seed=42)
    target, draft, toks, counts, ua, us = make_verify(T, 43, 6, 4, 50000)
    drawn, taken = T.zeros(6, 5, dtype=T.int32, device="cuda"), T.zeros(6, dtype=T.int32, device="cuda")
    pool = Pool(T, q3lib, "e4m3", 40, 4, 128)
    rows = T.randn(2, 640, 4 * 128, generator=_gen(T, 44), device="cuda")
    back = T.zeros_like(rows)
    slots = T.randperm(640, generator=_gen(T, 45), device="cuda").int()

    def verify(stream):
        q3lib.verify_drafts(drawn.data_ptr(), taken.data_ptr(), target.data_ptr(), target.stride(0),
                            target.stride(1), draft.data_ptr(), draft.stride(0), draft.stride(1),
                            toks.data_ptr(), counts.data_ptr(), ua.data_ptr(), us.data_ptr(), 6, 4, 50000,
                            stream)

    def move(stream):
        q3lib.kv_write(pool.handle, rows[0].data_ptr(), rows[1].data_ptr(), q3lib.TYPE_F32, 512, 512,
                       slots.data_ptr(), 640, stream)
        q3lib.kv_read(pool.handle, back[0].data_ptr(), back[1].data_ptr(), q3lib.TYPE_F32, 512, 512,
                      slots.data_ptr(), 640, stream)

    calls = [own.call, far.call, verify, move]
    results = [own.out_buf, far.out_buf, drawn, taken, back]
    for call in calls:
        call(None)
        T.cuda.synchronize()
    alone = [x.clone() for x in results]
    own.check()
    far.check()
    streams = [T.cuda.Stream() for _ in calls]

    def again():
        for x in results:
            x.fill_(9)
        T.cuda.synchronize()

    again()
    for _ in range(4):
        for call, s in zip(calls, streams):
            call(s.cuda_stream)
    T.cuda.synchronize()
    assert all(T.equal(x, y) for x, y in zip(results, alone))
    main, graph = T.cuda.Stream(), T.cuda.CUDAGraph()
    with T.cuda.graph(graph, stream=main):
        for call, s in zip(calls, streams):
            s.wait_stream(main)
            call(s.cuda_stream)
        for s in streams:
            main.wait_stream(s)
    again()
    graph.replay()
    T.cuda.synchronize()
    assert all(T.equal(x, y) for x, y in zip(results, alone))

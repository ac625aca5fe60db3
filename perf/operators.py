"""The serving operators over a paged KV pool, as cases that can be timed and compared.

Five operators, each in a plain form (elementary torch operations) and, where `own` is true, as the
calls a user makes of this library:

  write    a batch of new K/V rows goes into the pool, quantised to e4m3 (or stored as bf16)
  read     rows of the pool come back as fp32, bf16 or fp16
  attn     attention of each sequence's newest rows over its own pages
  prefix   the same for sequences that also share one prefix
  verify   drafted tokens accepted or rejected against the target's probabilities

The pool is [page][kv_head][16][head_dim] for K and for V. An e4m3 pool has one power of two for
each (token, head) row of K and of V: the value is code * 2^(byte - 127), and the byte is the
smallest for which the row's largest finite magnitude is at most 448 * 2^(byte - 127).
"""
import math
import os
import random
import sys

import torch

own = False

PAGE = 16
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # One decoded token's K and V rows: what every step of a single sequence writes per layer.
        dict(name="write 1 token", op="write", n=1, kv_heads=8, head_dim=128, pool="e4m3",
             type="f32", pad=0),
        # A prefill chunk's rows, columns of one [k;v] buffer (rows 2048 wide).
        dict(name="write 4096-token chunk", op="write", n=4096, kv_heads=8, head_dim=128,
             pool="e4m3", type="bf16", pad=1024),
        # A few odd rows of a narrow model read back.
        dict(name="read 37 rows", op="read", n=37, kv_heads=3, head_dim=64, pool="e4m3",
             type="f32", pad=5),
        # A whole 32768-token sequence read back, as a cache that moves to another place is.
        dict(name="read 32768 rows", op="read", n=32768, kv_heads=8, head_dim=128, pool="e4m3",
             type="bf16", pad=0),
        # Single-sequence decode at context 512: latency counts.
        dict(name="decode 1 x 512", op="attn", seqs=1, min_len=512, max_len=512, rows=1,
             kv_heads=8, group=2, head_dim=128, pool="e4m3", type="bf16"),
        # The batched decode configuration: 64 sequences of 128 to 4096 tokens.
        dict(name="decode 64 x 128-4096", op="attn", seqs=64, min_len=128, max_len=4096, rows=1,
             kv_heads=8, group=2, head_dim=128, pool="e4m3", type="bf16"),
        # Five rows a sequence (four drafts and the token before them), a bf16 pool.
        dict(name="drafts 16 x 5 x 100-5000", op="attn", seqs=16, min_len=100, max_len=5000, rows=5,
             kv_heads=8, group=2, head_dim=128, pool="bf16", type="bf16"),
        # A chat server: 64 conversations behind one 8192-token system prompt.
        dict(name="prefix 64 x 8192 + 1-600", op="prefix", seqs=64, min_len=1, max_len=600, rows=1,
             kv_heads=8, group=2, head_dim=128, pool="e4m3", type="bf16", prefix=8192),
        # A short ragged prefix in a bf16 pool, odd everywhere.
        dict(name="prefix 7 x 1003 + 0-77", op="prefix", seqs=7, min_len=0, max_len=77, rows=3,
             kv_heads=2, group=5, head_dim=64, pool="bf16", type="bf16", prefix=1003),
        # Many answers sampled from one long document, two rows each: matrix work.
        dict(name="prefix 256 x 2 x 32768", op="prefix", seqs=256, min_len=16, max_len=256, rows=2,
             kv_heads=8, group=4, head_dim=128, pool="e4m3", type="f16", prefix=32768),
        # One sequence's four drafts against the whole vocabulary.
        dict(name="verify 1 x 4 x 151936", op="verify", seqs=1, drafts=4, vocab=151936,
             one_hot=False),
        # A serving batch's drafts.
        dict(name="verify 64 x 5 x 151936", op="verify", seqs=64, drafts=5, vocab=151936,
             one_hot=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attn", "attn", "prefix", "prefix", "verify"])
    pool = rng.choice(["e4m3", "e4m3", "bf16"])
    head_dim = rng.choice([64, 128, 128])
    if op in ("write", "read"):
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        return dict(op=op, n=_log(rng, 1, (4096 if op == "write" else 32768) * 8 // max(8, kv_heads)),
                    kv_heads=kv_heads, head_dim=head_dim, pool=pool,
                    type=rng.choice(["f32", "bf16", "f16"]), pad=rng.choice([0, 1, 8, 24]))
    if op == "verify":
        return dict(op=op, seqs=_log(rng, 1, 64), drafts=rng.randint(0, 8),
                    vocab=_log(rng, 100, 151936), one_hot=rng.random() < 0.3)
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    rows = rng.choice([1, 1, 2, 4, 5, 8])
    typ = "bf16" if pool == "bf16" else rng.choice(["bf16", "f16"])
    if op == "attn":
        seqs = _log(rng, 1, 64)
        max_len = _log(rng, 1, min(32768, 262144 // seqs))
        return dict(op=op, seqs=seqs, min_len=rng.randint(0, max_len), max_len=max_len, rows=rows,
                    kv_heads=kv_heads, group=group, head_dim=head_dim, pool=pool, type=typ)
    seqs = _log(rng, 1, 256)
    max_len = _log(rng, 1, 600)
    most = 256 * 2 * 4 * 8 * 32768 // (seqs * rows * group * kv_heads)
    return dict(op=op, seqs=seqs, min_len=rng.randint(0, max_len), max_len=max_len, rows=rows,
                kv_heads=kv_heads, group=group, head_dim=head_dim, pool=pool, type=typ,
                prefix=_log(rng, 1, min(32768, most)))


def _lengths(case):
    """Every sequence's own length: spread evenly from min_len to max_len."""
    n, lo, hi = case["seqs"], case["min_len"], case["max_len"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _row_counts(case):
    """Every sequence's number of query rows: `rows`, and each third one fewer where there are more than one."""
    r = case["rows"]
    return [r - 1 if r > 1 and i % 3 == 2 else r for i in range(case["seqs"])]


def work(case):
    op = case["op"]
    if op == "verify":
        rows = 1 if case["one_hot"] or case["drafts"] == 0 else 2
        return {"bytes": case["seqs"] * (rows * case["vocab"] * 4 + case["drafts"] * 20 + 16),
                "flops": case["seqs"] * 3 * case["vocab"]}
    d, h = case["head_dim"], case["kv_heads"]
    cell = d + 1 if case["pool"] == "e4m3" else 2 * d  # bytes of one head's K or V row in the pool
    if op in ("write", "read"):
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": case["n"] * (2 * h * (size * d + cell) + 4), "flops": 4 * case["n"] * h * d}
    lens, rows = _lengths(case), _row_counts(case)
    keys = case.get("prefix", 0) + sum(lens)
    pairs = sum(r * (n + case.get("prefix", 0)) for r, n in zip(rows, lens))
    heads = h * case["group"]
    return {"bytes": 2 * h * cell * keys + 4 * heads * d * sum(rows) + 4 * (keys // PAGE),
            "flops": 4 * pairs * heads * d}


# ------------------------------------------------------------------ the pool in plain form

def _two_to(byte):
    """2^(byte - 127) of int32 bytes in [0, 254]."""
    f = (byte << 23).view(torch.float32)
    return torch.where(byte == 0, torch.full_like(f, 2.0 ** -127), f)


def _quantise(x):
    """fp32 rows [..., head_dim] -> (e4m3 codes, int32 bytes [...])."""
    big = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    part, e = torch.frexp(big)
    byte = torch.where(big > 0, (e + (127 - 9) + (part > 0.875)).clamp(0, 254), torch.zeros_like(e))
    scaled = x * ((254 - byte) << 23).view(torch.float32).unsqueeze(-1)
    return scaled.clamp(-448, 448).to(torch.float8_e4m3fn), byte


def _values(s, which, page, off):
    """fp32 rows [..., kv_heads, head_dim] of the pool at (page, offset in the page)."""
    rows = s[which][page, :, off]
    if s["case"]["pool"] == "bf16":
        return rows.float()
    return rows.view(torch.float8_e4m3fn).float() * _two_to(
        s["exps"][page, :, off, 0 if which == "k" else 1].int()).unsqueeze(-1)


def _new_pool(case, n_pages, g):
    """A pool of random rows, and one page behind it that nothing of the library's sees."""
    h, d = case["kv_heads"], case["head_dim"]
    s = {"case": case, "n_pages": n_pages}
    if case["pool"] == "e4m3":
        s["exps"] = torch.empty(n_pages + 1, h, PAGE, 2, dtype=torch.uint8, device=DEV)
    for i, which in enumerate("kv"):
        x = torch.randn(n_pages + 1, h, PAGE, d, generator=g, device=DEV)
        # Some heads and tokens are larger than others, as in a trained model's cache.
        x *= torch.exp2(torch.randint(-2, 2, (n_pages + 1, h, PAGE, 1), generator=g, device=DEV))
        if case["pool"] == "bf16":
            s[which] = x.to(torch.bfloat16)
        else:
            codes, byte = _quantise(x)
            s[which] = codes.view(torch.uint8)
            s["exps"][..., i] = byte.to(torch.uint8)
    return s


# ------------------------------------------------------------------ prepare

def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = case["op"]
    if op == "verify":
        s = _prepare_verify(case, g)
    elif op in ("write", "read"):
        s = _prepare_rows(case, g)
    else:
        s = _prepare_attn(case, g, seed)
    if own:
        _handles(s)
    return s


def _prepare_rows(case, g):
    n, h, d = case["n"], case["kv_heads"], case["head_dim"]
    n_pages = (n + n // 2 + PAGE) // PAGE + 1
    s = _new_pool(case, n_pages, g)
    s["slots"] = torch.randperm(n_pages * PAGE, generator=g, device=DEV)[:n].int()
    if n > 2:  # a padded batch: rows that belong to nothing
        s["slots"][n // 2] = -1
    # Rows lie `width` apart, as columns of a wider buffer.
    s["width"] = h * d + case["pad"]
    t = TYPES[case["type"]]
    for which in "kv":
        if case["op"] == "write":
            x = torch.randn(n, s["width"], generator=g, device=DEV)
            x *= torch.exp2(torch.randint(-3, 3, (n, 1), generator=g, device=DEV))
            s["in_" + which] = x.to(t)
        else:
            s["out_" + which] = torch.zeros(n, s["width"], dtype=t, device=DEV)
    return s


def _prepare_attn(case, g, seed):
    rng = random.Random(seed)
    lens, rows = _lengths(case), _row_counts(case)
    order = list(range(case["seqs"]))
    rng.shuffle(order)
    lens, rows = [lens[i] for i in order], [rows[i] for i in order]
    prefix = case.get("prefix", 0)
    width = max(1, -(-max(lens) // PAGE))
    own_pages = sum(-(-n // PAGE) for n in lens)
    prefix_pages = -(-prefix // PAGE)
    n_pages = own_pages + prefix_pages + 3
    s = _new_pool(case, n_pages, g)
    ids = torch.randperm(n_pages, generator=g, device=DEV).int()
    # Each sequence's pages in the order they were handed out; entries behind its last are unused.
    used = torch.tensor([-(-n // PAGE) for n in lens], device=DEV)
    at = torch.arange(width, device=DEV)
    first = torch.cumsum(used, 0) - used
    s["table"] = torch.where(at < used[:, None], ids[(first[:, None] + at).clamp(max=n_pages - 1)],
                             torch.full((), -1, dtype=torch.int32, device=DEV)).contiguous()
    s["prefix_table"] = ids[own_pages:own_pages + max(1, prefix_pages)].contiguous()
    s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["n_q"], s["n_heads"] = starts[-1], case["kv_heads"] * case["group"]
    t = TYPES[case["type"]]
    s["q"] = (2 * torch.randn(s["n_q"], s["n_heads"], case["head_dim"], generator=g, device=DEV)).to(t)
    s["out"] = torch.zeros_like(s["q"])
    return s


def _prepare_verify(case, g):
    b, k, v = case["seqs"], case["drafts"], case["vocab"]
    s = {"case": case}
    logits = 3 * torch.randn(b, k + 1, v, generator=g, device=DEV)
    s["target"] = _softmax(logits)
    if k:
        draft = _softmax(logits[:, :k] + 0.7 * torch.randn(b, k, v, generator=g, device=DEV))
        race = torch.empty(b, k, v, device=DEV).exponential_(generator=g)
        s["tokens"] = (draft / race).argmax(-1).int()
    else:
        draft = torch.zeros(b, 0, v, device=DEV)
        s["tokens"] = torch.zeros(b, 0, dtype=torch.int32, device=DEV)
    s["draft"] = None if case["one_hot"] else draft
    # Each third sequence has fewer drafts than the others.
    counts = [max(0, k - 1) if i % 3 == 2 else k for i in range(b)]
    s["n_drafts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
    s["u_accept"] = torch.rand(b, k, generator=g, device=DEV)
    s["u_sample"] = torch.rand(b, generator=g, device=DEV)
    s["out_tokens"] = torch.zeros(b, k + 1, dtype=torch.int32, device=DEV)
    s["out_accepted"] = torch.zeros(b, dtype=torch.int32, device=DEV)
    return s


def _softmax(x):
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


# ------------------------------------------------------------------ run

def run(s):
    op = s["case"]["op"]
    if own:
        return _own_run(s)
    if op == "write":
        return _plain_write(s)
    if op == "read":
        return _plain_read(s)
    if op == "verify":
        return _plain_verify(s)
    return _plain_attn(s)


def _pool_outputs(s):
    n = s["n_pages"]
    if s["case"]["pool"] == "bf16":
        return {"k": s["k"][:n], "v": s["v"][:n]}
    return {"k": s["k"][:n].view(torch.float8_e4m3fn), "v": s["v"][:n].view(torch.float8_e4m3fn),
            "exps": s["exps"][:n]}


def _plain_write(s):
    case = s["case"]
    n, h, d = case["n"], case["kv_heads"], case["head_dim"]
    slots = s["slots"].long()
    slots = torch.where(slots < 0, s["n_pages"] * PAGE, slots)  # nothing's rows go behind the pool
    page, off = slots // PAGE, slots % PAGE
    for i, which in enumerate("kv"):
        x = s["in_" + which][:, :h * d].reshape(n, h, d).float()
        if case["pool"] == "bf16":
            s[which][page, :, off] = x.to(torch.bfloat16)
        else:
            codes, byte = _quantise(x)
            s[which][page, :, off] = codes.view(torch.uint8)
            s["exps"][page, :, off, i] = byte.to(torch.uint8)
    return _pool_outputs(s)


def _plain_read(s):
    case = s["case"]
    n, h, d = case["n"], case["kv_heads"], case["head_dim"]
    slots = s["slots"].long()
    page, off = slots.clamp(min=0) // PAGE, slots.clamp(min=0) % PAGE
    for which in "kv":
        x = _values(s, which, page, off) * (slots >= 0)[:, None, None]
        s["out_" + which][:, :h * d] = x.reshape(n, h * d).to(TYPES[case["type"]])
    return {"k": s["out_k"], "v": s["out_v"]}


def _plain_attn(s):
    case = s["case"]
    h, grp, d, b = case["kv_heads"], case["group"], case["head_dim"], case["seqs"]
    prefix, rows = case.get("prefix", 0), case["rows"]
    scale = 1.0 / math.sqrt(d)
    q = s["q"].float().view(s["n_q"], h, grp, d)
    lens, starts = s["kv_len"].long(), s["q_start"].long()
    counts = starts[1:] - starts[:-1]
    # The queries of each sequence, padded to `rows`.
    i = torch.arange(rows, device=DEV)
    at = (starts[:-1, None] + i).clamp(max=s["n_q"] - 1)
    qb = q[at]                                                        # [b, rows, h, grp, d]
    width = s["table"].shape[1] * PAGE
    key = torch.arange(width, device=DEV)
    page = s["table"].long().clamp(min=0)[:, key // PAGE]             # [b, width]
    there = key < lens[:, None]
    k = _values(s, "k", page, (key % PAGE).expand(b, -1))              # [b, width, h, d]
    v = _values(s, "v", page, (key % PAGE).expand(b, -1)) * there[:, :, None, None]
    pos = lens[:, None] - counts[:, None] + i                         # [b, rows]
    seen = key <= pos[:, :, None]
    t = torch.einsum("brhgd,bkhd->brhgk", qb, k) * scale
    t = torch.where((seen & there[:, None])[:, :, None, None], t, -math.inf)
    del k
    m = t.amax(-1)
    if prefix:
        at_p = torch.arange(prefix, device=DEV)
        pp = s["prefix_table"].long()[at_p // PAGE]
        kp, vp = _values(s, "k", pp, at_p % PAGE), _values(s, "v", pp, at_p % PAGE)
        tp = torch.einsum("nhgd,khd->nhgk", q, kp) * scale            # once for all rows
        m_p = tp.amax(-1)
        e_p = torch.exp(tp - m_p[..., None])
        del tp
        l_p, o_p = e_p.sum(-1), torch.einsum("nhgk,khd->nhgd", e_p, vp)
        del e_p
        m_p, l_p, o_p = m_p[at], l_p[at], o_p[at]
        m_all = torch.maximum(m, m_p)
    else:
        m_all = m
    m_safe = torch.where(m_all == -math.inf, torch.zeros_like(m_all), m_all)
    e = torch.exp(t - m_safe[..., None])
    del t
    l, o = e.sum(-1), torch.einsum("brhgk,bkhd->brhgd", e, v)
    if prefix:
        f = torch.exp(m_p - m_all)
        l, o = l + l_p * f, o + o_p * f[..., None]
    o = torch.where(l[..., None] > 0, o / l[..., None], torch.zeros_like(o))
    # Back to the rows; the padding goes to a row behind the last.
    to = torch.where(i < counts[:, None], starts[:-1, None] + i, s["n_q"]).reshape(-1)
    out = torch.zeros(s["n_q"] + 1, h * grp, d, dtype=s["q"].dtype, device=DEV)
    out[to] = o.reshape(b * rows, h * grp, d).to(s["q"].dtype)
    return out[:-1]


def _plain_verify(s):
    case = s["case"]
    b, k, v = case["seqs"], case["drafts"], case["vocab"]
    rows = torch.arange(b, device=DEV)
    counts, tok = s["n_drafts"].long(), s["tokens"].long()
    p_tok = s["target"][:, :k].gather(2, tok[..., None])[..., 0].double()
    if s["draft"] is None:
        q_tok = torch.ones_like(p_tok)
    else:
        q_tok = s["draft"].gather(2, tok[..., None])[..., 0].double()
    j = torch.arange(k, device=DEV)
    good = (s["u_accept"].double() * q_tok < p_tok) & (j < counts[:, None])
    accepted = torch.cumprod(good.long(), 1).sum(1)
    p = s["target"][rows, accepted].double()
    if k:
        row = accepted.clamp(max=k - 1)
        if s["draft"] is None:
            q = torch.zeros_like(p).scatter_(1, tok[rows, row][:, None], 1.0)
        else:
            q = s["draft"][rows, row].double()
        q = q * (accepted < counts)[:, None]
    else:
        q = torch.zeros_like(p)
    r = (p - q).clamp(min=0)
    # A residual with nothing in it leaves the target's own probabilities.
    r = torch.where(r.sum(1, keepdim=True) > 0, r, p)
    c = torch.cumsum(r, 1)
    over = c > s["u_sample"].double()[:, None] * c[:, -1:]
    token = torch.where(over.any(1), over.int().argmax(1), v - 1)
    at = torch.arange(k + 1, device=DEV)
    padded = torch.cat([tok, torch.zeros(b, 1, dtype=torch.long, device=DEV)], 1)
    out = torch.where(at < accepted[:, None], padded, torch.full_like(padded, -1))
    out = torch.where(at == accepted[:, None], token[:, None], out)
    return {"tokens": out.int(), "accepted": accepted.int()}


# ------------------------------------------------------------------ the library's calls

def _library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3.cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import q3b200
    return q3b200


def _handles(s):
    """What a user's program keeps beside its buffers: the pool's description and the workspace."""
    q3, case = _library(), s["case"]
    s["q3"] = q3
    if case["op"] == "verify":
        return
    types = {"f32": q3.TYPE_F32, "bf16": q3.TYPE_BF16, "f16": q3.TYPE_F16, "e4m3": q3.TYPE_E4M3}
    s["type"] = types[case["type"]]
    s["pool"] = q3.KvPool(s["k"].data_ptr(), s["v"].data_ptr(),
                          s["exps"].data_ptr() if "exps" in s else None, s["n_pages"],
                          case["kv_heads"], case["head_dim"], types[case["pool"]])
    if case["op"] in ("attn", "prefix"):
        size = q3.paged_attn_workspace_size(s["pool"], s["n_heads"], s["n_q"], case["seqs"],
                                            case["rows"], case.get("prefix", 0))
        s["ws"] = torch.empty(size, dtype=torch.uint8, device=DEV)


def _own_run(s):
    case, q3 = s["case"], s["q3"]
    op = case["op"]
    if op == "write":
        q3.kv_write(s["pool"], s["in_k"].data_ptr(), s["in_v"].data_ptr(), s["type"], s["width"],
                    s["width"], s["slots"].data_ptr(), case["n"])
        return _pool_outputs(s)
    if op == "read":
        q3.kv_read(s["pool"], s["out_k"].data_ptr(), s["out_v"].data_ptr(), s["type"], s["width"],
                   s["width"], s["slots"].data_ptr(), case["n"])
        return {"k": s["out_k"], "v": s["out_v"]}
    if op == "verify":
        k, v = case["drafts"], case["vocab"]
        q3.verify_drafts(s["out_tokens"].data_ptr(), s["out_accepted"].data_ptr(),
                         s["target"].data_ptr(), (k + 1) * v, v,
                         s["draft"].data_ptr() if k and s["draft"] is not None else None, k * v, v,
                         s["tokens"].data_ptr() if k else None, s["n_drafts"].data_ptr(),
                         s["u_accept"].data_ptr() if k else None, s["u_sample"].data_ptr(),
                         case["seqs"], k, v)
        return {"tokens": s["out_tokens"], "accepted": s["out_accepted"]}
    width = s["n_heads"] * case["head_dim"]
    if op == "attn":
        q3.paged_attn(s["out"].data_ptr(), s["ws"].data_ptr(), s["q"].data_ptr(), s["type"], width,
                      width, s["pool"], s["n_heads"], s["n_q"], case["seqs"], case["rows"],
                      s["q_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(),
                      s["table"].shape[1])
    else:
        q3.prefix_attn(s["out"].data_ptr(), s["ws"].data_ptr(), s["q"].data_ptr(), s["type"], width,
                       width, s["pool"], s["n_heads"], s["n_q"], case["seqs"], case["rows"],
                       s["q_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(),
                       s["table"].shape[1], s["prefix_table"].data_ptr(), case["prefix"])
    return s["out"]


# ------------------------------------------------------------------ exact, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "write":
        return _exact_write(s)
    if op == "read":
        return _exact_read(s)
    if op == "verify":
        return _exact_verify(s)
    return _exact_attn(s)


def _exact_write(s):
    case = s["case"]
    h, d = case["kv_heads"], case["head_dim"]
    to = s["slots"] >= 0
    slots = s["slots"][to].long()
    got = {}
    for i, which in enumerate("kv"):
        flat = s[which][:s["n_pages"]].transpose(1, 2).reshape(-1, h, d)
        x = s["in_" + which][to][:, :h * d].reshape(-1, h, d).double()
        if case["pool"] == "bf16":
            pool = flat.double()
            pool[slots] = x
        else:
            big = x.abs().amax(-1)
            e = torch.ceil(torch.log2(big / 448))
            e = torch.where(big <= 448 * torch.exp2(e - 1), e - 1, e)
            e = torch.where(big > 448 * torch.exp2(e), e + 1, e).clamp(min=-127)
            y = x / torch.exp2(e)[..., None]
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            pool = flat.view(torch.float8_e4m3fn).double()
            pool[slots] = torch.round(y / step) * step
            exps = got.setdefault("exps", s["exps"][:s["n_pages"]].transpose(1, 2).reshape(-1, h, 2).clone())
            exps[slots, :, i] = (e + 127).to(torch.uint8)
        got[which] = pool.view(s["n_pages"], PAGE, h, d).transpose(1, 2)
    if "exps" in got:
        got["exps"] = got["exps"].view(s["n_pages"], PAGE, h, 2).transpose(1, 2)
    return got


def _exact_rows(s, which, slots):
    """[len(slots), kv_heads, head_dim] in 64 bits."""
    h, d = s["case"]["kv_heads"], s["case"]["head_dim"]
    page, off = torch.div(slots, PAGE, rounding_mode="floor"), slots % PAGE
    rows = s[which].permute(0, 2, 1, 3)[page, off]
    if s["case"]["pool"] == "bf16":
        return rows.double()
    e = s["exps"].permute(0, 2, 1, 3)[page, off][..., 0 if which == "k" else 1].double() - 127
    return rows.view(torch.float8_e4m3fn).double() * torch.exp2(e)[..., None]


def _exact_read(s):
    case = s["case"]
    h, d = case["kv_heads"], case["head_dim"]
    got = {}
    for which in "kv":
        out = s["out_" + which].double()
        to = s["slots"] >= 0
        out[to, :h * d] = _exact_rows(s, which, s["slots"][to].long()).flatten(1)
        got[which] = out
    return got


def _exact_attn(s):
    case = s["case"]
    h, grp, d = case["kv_heads"], case["group"], case["head_dim"]
    prefix = case.get("prefix", 0)
    lens, starts = s["kv_len"].tolist(), s["q_start"].tolist()
    slots = lambda table, n: (table.long()[torch.arange(n, device=DEV) // PAGE] * PAGE  # noqa: E731
                              + torch.arange(n, device=DEV) % PAGE)
    out = torch.zeros(s["n_q"], h * grp, d, dtype=torch.float64, device=DEV)
    shared = [_exact_rows(s, w, slots(s["prefix_table"], prefix)) for w in "kv"]
    for b, n in enumerate(lens):
        k, v = (torch.cat([a, _exact_rows(s, w, slots(s["table"][b], n))])
                for a, w in zip(shared, "kv"))
        count = starts[b + 1] - starts[b]
        q = s["q"][starts[b]:starts[b + 1]].double().view(count, h, grp, d)
        for i in range(count):
            # Row i is the sequence's token n - count + i: it sees the prefix and its own up to itself.
            most = prefix + max(0, n - count + i + 1)
            if not most:
                continue
            t = (q[i].view(h, grp, d) @ k[:most].permute(1, 2, 0)) / math.sqrt(d)
            out[starts[b] + i] = (torch.softmax(t, -1) @ v[:most].transpose(0, 1)).reshape(h * grp, d)
    return out


def _exact_verify(s):
    case = s["case"]
    k = case["drafts"]
    tokens, taken = [], []
    for b in range(case["seqs"]):
        n = 0
        count = int(s["n_drafts"][b])
        while n < count:
            t = int(s["tokens"][b, n])
            q = 1.0 if s["draft"] is None else float(s["draft"][b, n, t])
            if not float(s["u_accept"][b, n]) * q < float(s["target"][b, n, t]):
                break
            n += 1
        r = p = s["target"][b, n].double()
        if n < count and s["draft"] is None:
            r = p.clone()
            r[int(s["tokens"][b, n])] = max(0.0, float(r[int(s["tokens"][b, n])]) - 1.0)
        elif n < count:
            r = torch.relu(p - s["draft"][b, n].double())
        if float(r.sum()) <= 0:
            r = p
        sums = r.cumsum(0)
        at = int(torch.searchsorted(sums, float(s["u_sample"][b]) * sums[-1:], right=True)[0])
        tokens.append(s["tokens"][b, :n].tolist() + [min(at, case["vocab"] - 1)] + [-1] * (k - n))
        taken.append(n)
    return {"tokens": torch.tensor(tokens, dtype=torch.int32),
            "accepted": torch.tensor(taken, dtype=torch.int32)}

"""Arguments that the paged-pool operators refuse before they touch a GPU."""
import ctypes as C

import pytest

P = 1 << 20  # an address that is never read: every call here is refused first


def _pool(q3, **over):
    f = dict(k=P, v=P, exps=P, n_pages=4, n_kv_heads=2, head_dim=128, type=q3.TYPE_E4M3)
    f.update(over)
    return q3.KvPool(*(f[n] for n, _ in q3.KvPool._fields_))


BAD_POOLS = [dict(type=0), dict(type=2), dict(type=7), dict(head_dim=0), dict(head_dim=96),
             dict(head_dim=256), dict(n_kv_heads=0), dict(n_kv_heads=-1), dict(n_pages=0),
             dict(n_pages=1 << 27), dict(k=None), dict(v=None), dict(exps=None), dict(k=P + 8),
             dict(v=P + 4), dict(exps=P + 1), dict(type=1)]


@pytest.mark.parametrize("over", BAD_POOLS, ids=str)
def test_bad_pools_are_refused(q3lib, over):
    pool = _pool(q3lib, **over)
    with pytest.raises(q3lib.InvalidArgument, match="KV pool"):
        q3lib.kv_write(pool, P, P, q3lib.TYPE_F32, 256, 256, P, 1)
    with pytest.raises(q3lib.InvalidArgument, match="KV pool"):
        q3lib.kv_read(pool, P, P, q3lib.TYPE_F32, 256, 256, P, 1)
    with pytest.raises(q3lib.InvalidArgument, match="KV pool"):
        q3lib.paged_attn(P, P, P, q3lib.TYPE_BF16, 512, 512, pool, 4, 1, 1, 1, P, P, P, 4)


def test_null_pool_is_refused(q3lib):
    L = q3lib.lib()
    assert L.q3_kv_write(None, P, P, 0, 256, 256, P, 1, None) == 2
    assert L.q3_kv_read(None, P, P, 0, 256, 256, P, 1, None) == 2
    assert L.q3_paged_attn_workspace_size(None, 4, 1, 1, 1, 0) == 0


@pytest.mark.parametrize("over", [dict(type=3), dict(type=-1), dict(n=-1), dict(k=None), dict(v=None),
                                  dict(slots=None), dict(k_stride=255), dict(v_stride=0),
                                  dict(k=P + 2), dict(slots=P + 2)], ids=str)
def test_bad_rows_are_refused(q3lib, over):
    f = dict(k=P, v=P, type=q3lib.TYPE_F32, k_stride=256, v_stride=256, slots=P, n=1)
    f.update(over)
    for call in (q3lib.kv_write, q3lib.kv_read):
        with pytest.raises(q3lib.InvalidArgument, match="KV rows"):
            call(_pool(q3lib), *f.values())


def test_no_rows_is_no_call(q3lib):
    q3lib.kv_write(_pool(q3lib), None, None, q3lib.TYPE_F32, 256, 256, None, 0)
    q3lib.kv_read(_pool(q3lib), None, None, q3lib.TYPE_F32, 256, 256, None, 0)


ATTN = dict(out=P, ws=P, q=P, type=1, q_stride=512, out_stride=512, n_heads=4, n_q=3, n_seqs=2,
            max_q=2, q_start=P, kv_len=P, table=P, table_stride=4, prefix_table=P, prefix_len=20)


def _attn(q3, pool, prefix, **over):
    f = dict(ATTN)
    f.update(over)
    last = [f.pop("prefix_table"), f.pop("prefix_len")]
    args = list(f.values())
    args.insert(6, pool)
    (q3.prefix_attn if prefix else q3.paged_attn)(*args, *(last if prefix else []))


@pytest.mark.parametrize("over", [
    dict(type=0), dict(type=3), dict(n_heads=0), dict(n_heads=3), dict(n_heads=130), dict(n_q=-1),
    dict(n_seqs=-1), dict(max_q=0), dict(max_q=65), dict(table_stride=-1), dict(table_stride=(1 << 26) + 1), dict(out=None),
    dict(ws=None), dict(q=None), dict(q_start=None), dict(kv_len=None), dict(table=None),
    dict(q_stride=511), dict(q_stride=516), dict(out_stride=508), dict(q=P + 8), dict(out=P + 2),
    dict(ws=P + 4), dict(q_start=P + 1), dict(table=P + 2)], ids=str)
def test_bad_attention_is_refused(q3lib, over):
    for prefix in (False, True):
        with pytest.raises(q3lib.InvalidArgument, match="paged attention"):
            _attn(q3lib, _pool(q3lib), prefix, **over)


def test_bad_prefix_is_refused(q3lib):
    for over in (dict(prefix_len=-1), dict(prefix_len=(1 << 28) + 1), dict(prefix_table=None),
                 dict(prefix_table=P + 2)):
        with pytest.raises(q3lib.InvalidArgument, match="paged attention"):
            _attn(q3lib, _pool(q3lib), True, **over)


def test_fp16_rows_need_an_e4m3_pool(q3lib):
    with pytest.raises(q3lib.InvalidArgument, match="paged attention"):
        _attn(q3lib, _pool(q3lib, type=q3lib.TYPE_BF16, exps=None), False, type=q3lib.TYPE_F16)


def test_no_attention_rows_is_no_call(q3lib):
    _attn(q3lib, _pool(q3lib), False, n_q=0)
    _attn(q3lib, _pool(q3lib), True, n_seqs=0, out=None)


def test_workspace_size(q3lib):
    pool = _pool(q3lib)
    assert q3lib.paged_attn_workspace_size(pool, 4, 3, 2, 2, 0) > 0
    assert (q3lib.paged_attn_workspace_size(pool, 4, 3, 2, 2, 1 << 15)
            >= q3lib.paged_attn_workspace_size(pool, 4, 3, 2, 2, 0))
    for bad in ((3, 3, 2, 2, 0), (4, -1, 2, 2, 0), (4, 3, -1, 2, 0), (4, 3, 2, 0, 0), (4, 3, 2, 2, -1)):
        assert q3lib.paged_attn_workspace_size(pool, *bad) == 0


VERIFY = dict(tokens=P, n_accepted=P, target=P, t_seq=300, t_row=100, draft=P, d_seq=200, d_row=100,
              draft_tokens=P, n_drafts=P, u_accept=P, u_sample=P, n_seqs=2, max_drafts=2, vocab=100)


@pytest.mark.parametrize("over", [
    dict(n_seqs=-1), dict(max_drafts=-1), dict(max_drafts=1025), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(tokens=None),
    dict(n_accepted=None), dict(target=None), dict(draft_tokens=None), dict(u_accept=None),
    dict(u_sample=None), dict(t_row=99), dict(d_row=99), dict(t_seq=-1), dict(d_seq=-1),
    dict(target=P + 2), dict(tokens=P + 1)], ids=str)
def test_bad_verification_is_refused(q3lib, over):
    f = dict(VERIFY)
    f.update(over)
    with pytest.raises(q3lib.InvalidArgument, match="draft verification"):
        q3lib.verify_drafts(*f.values())


def test_no_sequences_is_no_call(q3lib):
    q3lib.verify_drafts(*dict(VERIFY, n_seqs=0).values())


def test_a_refusal_leaves_its_message(q3lib):
    assert q3lib.lib().q3_kv_write(C.byref(_pool(q3lib)), P, P, 9, 256, 256, P, 1, None) == 2
    assert b"type must be F32" in q3lib.lib().q3_last_error()

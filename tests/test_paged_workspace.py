"""The workspace of paged attention serves every smaller call."""
import pytest

P = 1 << 20


def _pool(q3, h, d, e4m3):
    return q3.KvPool(P, P, P if e4m3 else None, 4, h, d, q3.TYPE_E4M3 if e4m3 else q3.TYPE_BF16)


@pytest.mark.parametrize("h,group,d", [(8, 2, 128), (1, 8, 64), (2, 64, 128), (16, 1, 128), (37, 3, 64)])
@pytest.mark.parametrize("e4m3", [True, False])
def test_size_never_falls(q3lib, h, group, d, e4m3):
    pool = _pool(q3lib, h, d, e4m3)

    def size(n_q, n_seqs=4, max_q=1, prefix=0):
        return q3lib.paged_attn_workspace_size(pool, h * group, n_q, n_seqs, max_q, prefix)

    rows = sorted(set(range(0, 300)) | {x for n in range(9, 13) for x in range(2 ** n - 3, 2 ** n + 4)})
    for prefix in (0, 1, 200, 2304, 2432, 8192, 32768, 1 << 28):
        sizes = [size(n, prefix=prefix) for n in rows]
        assert sizes == sorted(sizes) and sizes[0] > 0
    lengths = sorted(set(range(0, 9000, 61)) | {2304, 2432} | {2 ** n + x for n in range(13, 29) for x in (-1, 0)})
    for n_q in (1, 63, 64, 65, 128, 129, 1000):
        sizes = [size(n_q, prefix=p) for p in lengths]
        assert sizes == sorted(sizes) and sizes[0] > 0
    most = 128 // group
    for prefix in (0, 2304):
        sizes = [size(128, max_q=m, prefix=prefix) for m in range(1, most + 1)]
        assert sizes == sorted(sizes) and sizes[0] > 0
        sizes = [size(128, n_seqs=n, prefix=prefix) for n in (0, 1, 64, 128)]
        assert sizes == sorted(sizes)


def test_size_of_the_largest_batch(q3lib):
    """The most rows that the calls take."""
    pool = _pool(q3lib, 1, 64, True)
    assert (q3lib.paged_attn_workspace_size(pool, 1, 1 << 23, 1 << 23, 1, 4096)
            >= q3lib.paged_attn_workspace_size(pool, 1, 1 << 22, 1 << 22, 1, 4096) > 0)

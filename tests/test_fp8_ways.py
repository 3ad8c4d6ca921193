"""Which kernel an FP8 product takes at the sizes of the GPU tests, on a chip of 256 CUs: each of them is reached, dense and over groups, and K long enough for what each does along it."""
from tests import test_gpu_fp8_block as block
from tests import test_gpu_fp8_ways as more
from tests.gpu_util import hooks_lib

ROWS, TILES = ("rows 16x16", "rows 64x16", "rows 16x32", "rows 32x32", "rows 32x64"), ("tile 128x128", "tile 256x128", "tile 256x256")


def _way(m, n, k, groups=0, workspace=1):
    v = hooks_lib().cmx_debug_fp8_way(m, n, k, groups, workspace, 256)
    return (ROWS + TILES)[v & 255], v >> 8


def _most_blocks(ways):
    most = {}
    for way, k in ways:
        most[way] = max(most.get(way, 0), -(-k // 128))
    return most


def test_dense_sizes_take_every_kernel():
    most = _most_blocks((_way(*s), s[2]) for s in block.SHAPES + block.WAYS + more.DENSE)
    assert {w for w, parts in most if parts == 1} == set(ROWS + TILES)
    # two changes of the span whose scales lie in LDS
    assert all(most[w, 1] > 16 for w in TILES)
    assert any(parts > 1 for w, parts in most if w == TILES[0]) and all(parts == 1 for w, parts in most if w != TILES[0])


def test_groups_take_every_kernel():
    total = lambda sizes: sum(max(0, s) for s in sizes)
    for extra in (0, 37):
        most = _most_blocks((_way(total(s) + extra, n, k, len(s)), k) for s, n, k in block.GROUPS + more.GROUPED)
        assert set(most) == {(w, 1) for w in ROWS + TILES}
        assert all(most[w, 1] > 16 for w in TILES)


def test_only_a_call_with_a_workspace_is_shared_out():
    assert _way(250, 4100, 7184)[1] > 1 and _way(250, 4100, 7184, workspace=0)[1] == 1

"""How the attention over a cache is split, as its workspace query tells, without a GPU."""
import pytest


@pytest.mark.parametrize("B,T,H,G,D,page,blocks,window,splits", [
    (3, 1, 2, 16, 64, 16, 94, -1, 24), (520, 1, 1, 1, 64, 16, 94, -1, 3), (150, 1, 2, 1, 64, 32, 47, 1000, 3),
    (2, 1, 3, 1, 128, 64, 24, 1300, 21), (3, 9, 2, 2, 64, 32, 47, -1, 24)])
def test_sizes_that_are_split(B, T, H, G, D, page, blocks, window, splits):
    """A partial row: D means, a maximum and a total, eight rows a tile."""
    from neuratensor_b200 import build, native
    build.build()
    tiles = B * H * -(-T * G // 8)
    need = native.load().nt_kv_attention_workspace_bytes(B, T, H * G, H, D, page, blocks, window)
    assert need == tiles * splits * 8 * (D + 2) * 4

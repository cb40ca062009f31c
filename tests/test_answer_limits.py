"""hmx_linear_mx4 refuses what its launches' grids cannot hold before anything is enqueued (no GPU needed): past the limits it
is EINVAL, at them the call goes on to the workspace, which is missing."""
import pytest

from generative_recommenders_amd import hmx

P = 0x1000                  # a 16-byte aligned non-null address that a refused call never reads
EINVAL, EWORKSPACE = -1, -2


@pytest.mark.parametrize("kind,M,K,code", [
    (0, 655350, 160, EWORKSPACE), (0, 655351, 160, EINVAL), (1, 1048560, 160, EWORKSPACE), (1, 1048561, 160, EINVAL),
    (2, 1048560, 160, EWORKSPACE), (2, 1048561, 160, EINVAL), (0, 1048561, 64, EINVAL),
    # the threads that lay x out: tiles of 16 rows (fp32: 5) times pairs of 128 columns times 512 (mx8: 256)
    (1, 16, (1 << 23) * 8, EWORKSPACE), (1, 32 * 16, (1 << 23) * 8, EINVAL), (1, 31 * 16, (1 << 23) * 8, EWORKSPACE),
    (2, 63 * 16, (1 << 23) * 8, EWORKSPACE), (2, 64 * 16, (1 << 23) * 8, EINVAL), (0, 31 * 5, (1 << 23) * 8, EWORKSPACE),
    (0, 31 * 5 + 1, (1 << 23) * 8, EINVAL), (1, 1048560, 1 << 16, EINVAL)])
def test_linear_mx4_grids(kind, M, K, code):
    xs = P if kind == 2 else None
    assert hmx.lib().hmx_linear_mx4(P, K, xs, kind, M, P, P, 64, K, 0, P, None, 0, None) == code

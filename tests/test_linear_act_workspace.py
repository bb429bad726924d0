"""What gn_linear_act_workspace_bytes has room for (no GPU needed)."""
import pytest

gn = pytest.importorskip("gn_bwd")


def up(n, m):
    return (n + m - 1) // m * m


def layout(M, N, K):
    """The backward's operands laid out: dY, W and A in bf16, dW and db in fp32."""
    Np, Kp = up(N, 8), up(K, 8)
    return sum(up(n, 16) for n in (M * Np * 2, Np * Kp * 2, M * Kp * 2, Np * Kp * 4, Np * 4))


@pytest.mark.parametrize("M,N,K", [(8192, 1027, 1031), (8192, 2047, 1023), (8192, 513, 519), (8192, 767, 769)])
def test_odd_sizes_have_room_for_the_weight_gradients_planes(M, N, K):
    lib = gn.lib()
    planes = lib.gn_linear_workspace_bytes(M, up(N, 8), up(K, 8), gn.BF16)
    assert lib.gn_linear_workspace_bytes(M, N, K, gn.BF16) == 0 and planes > 0
    assert lib.gn_linear_act_workspace_bytes(M, N, K, gn.BF16) >= layout(M, N, K) + planes


def test_multiples_of_8_leave_them_to_the_linear_layers_query():
    assert gn.lib().gn_linear_act_workspace_bytes(8192, 1032, 1032, gn.BF16) == layout(8192, 1032, 1032)

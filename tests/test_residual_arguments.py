"""Arguments of the residual branch's and dropout's Python entries, in front of any call of the library."""
import pytest

torch = pytest.importorskip("torch")
gn = pytest.importorskip("gn_bwd")


def test_a_gate_without_rows_is_refused():
    """It would be taken for no gate."""
    h = torch.zeros(4, 8)
    args = dict(post="none", post_w=None, post_b=None, pre="none", pre_w=None, pre_b=None, scale=1.0, res_scale=1.0, p=0.0, seed=0,
                stream=0, step=0, post_eps=None, pre_eps=None, dev=0)
    with pytest.raises(gn.GnError, match="gate must have a row"):
        gn._branch(h, h, gate=torch.zeros(0, 8), **args)
    assert gn._branch(h, h, gate=None, **args).gates == 0


def test_numbers_of_numpy():
    """Seeds, places and steps drawn by numpy are the same numbers."""
    np = pytest.importorskip("numpy")
    gb = pytest.importorskip("grilly_bridge")
    for n in (np.int64(-7), np.uint64(2 ** 63 + 5), np.int32(9), np.uint8(200)):
        r, s = gn._rng(n, n, n, 0), gn._rng(int(n), int(n), int(n), 0)
        assert (r.seed, r.stream, r.step) == (s.seed, s.stream, s.step) == (int(n) % 2 ** 64,) * 3
        assert gb.dropout_params(0.1, n, n, n) == gb.dropout_params(0.1, int(n), int(n), int(n))
        assert gb.residual_norm_params(p=0.1, seed=n, stream=n, step=n) == gb.residual_norm_params(p=0.1, seed=int(n), stream=int(n), step=int(n))


@pytest.mark.gpu
def test_a_gate_without_rows_is_refused_by_both(gpu):
    h = torch.zeros(4, 8, device=gpu)
    gate = torch.zeros(0, 8, device=gpu)
    with pytest.raises(gn.GnError, match="gate must have a row"):
        gn.residual_norm_fwd(h, h, gate=gate)
    with pytest.raises(gn.GnError, match="gate must have a row"):
        gn.residual_norm_bwd(h, None, h, h, gate=gate)
    y, _ = gn.residual_norm_fwd(h[:0], h[:0], gate=gate)
    assert y.shape == (0, 8)

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

"""Options of SiT for fine patch grids (rotary, key_blocks, act8): what the constructors and setters refuse, and that a model without them
is what it was."""
import pytest
import torch

KW = dict(dim=96, depth=1, heads=1, mlp_dim=128, num_patches=10, num_vertices=3, num_channels=2)


@pytest.fixture(scope="module")
def mods():
    import sitk  # noqa: F401
    from sitk.models import sit
    from sitk.runtime import SitkError
    return sit, SitkError


@pytest.mark.parametrize("bad", [dict(rotary=()), dict(rotary=(33,)), dict(rotary=(-1, 4)), dict(rotary=(1, 1, 1, 1, 1)), dict(rotary=(0, 0)),
                                 dict(rotary=(4, 4), rotary_base=0.0), dict(rotary=(4,), rotary_base=float("inf")),
                                 dict(key_blocks=(96, 4)), dict(key_blocks=(0, 4)), dict(key_blocks=(2048, 4)), dict(key_blocks=(64, 0)),
                                 dict(key_blocks=(64,))])
def test_constructor_refuses(mods, bad):
    sit, SitkError = mods
    with pytest.raises(SitkError, match="rotary|key_blocks"):
        sit.SiT(**KW, **bad)


def test_positions_are_checked(mods):
    sit, SitkError = mods
    m = sit.SiT(**KW, rotary=(4, 4, 4))
    for bad in (torch.zeros(9, 3), torch.zeros(11, 3), torch.zeros(10, 2), torch.zeros(10), torch.zeros(2, 10, 3)):
        with pytest.raises(SitkError, match="positions"):
            m.set_patch_positions(bad)
    with pytest.raises(SitkError, match="not set"):
        m.transformer._rotary_inputs(11, "cpu")
    given = torch.randn(10, 3)
    m.set_patch_positions(given)
    pos, freqs = m.transformer._rotary_inputs(11, "cpu")
    assert pos.shape == (11, 3) and not pos[0].any() and torch.equal(pos[1:], given) and freqs.shape == (12,) and freqs.dtype == torch.float64
    given.zero_()                                             # the model keeps its own copy
    assert m.transformer._rotary_inputs(11, "cpu")[0].any()
    with pytest.raises(SitkError, match="11 tokens"):
        m.transformer._rotary_inputs(12, "cpu")
    for kind, kept in ((torch.float16, torch.float32), (torch.int16, torch.int64), (torch.float64, torch.float64)):
        m.set_patch_positions(torch.ones(10, 3, dtype=kind))
        assert m.transformer._rotary_inputs(11, "cpu")[0].dtype == kept
    with pytest.raises(SitkError, match="rotary=None"):
        sit.SiT(**KW).set_patch_positions(torch.zeros(10, 3))


def test_defaults_and_state_dict_are_unchanged(mods):
    sit, _ = mods
    plain, full = sit.SiT(**KW), sit.SiT(**KW, rotary=(4, 4, 4), key_blocks=(64, 2), act8=True)
    full.set_patch_positions(torch.zeros(10, 3))
    assert plain.transformer.fused_ok() and not full.transformer.fused_ok()
    assert set(plain.state_dict()) == set(full.state_dict())
    for opt in (dict(rotary=(4,)), dict(key_blocks=(64, 1)), dict(act8=True)):
        assert not sit.SiT(**KW, **opt).transformer.fused_ok()


def test_positions_of_a_captured_graph_stay(mods, monkeypatch):
    """Whatever a forward pass took under capture lives as long as the model (a replay reads it), also behind set_positions; passes outside a
    capture keep nothing, and positions that are not on the device cannot be brought there under capture."""
    import weakref
    sit, SitkError = mods
    t = sit.SiT(**KW, rotary=(4, 4, 4)).transformer
    t.set_positions(torch.randn(11, 3))
    monkeypatch.setattr(sit, "_capturing", lambda device: True)
    with pytest.raises(SitkError, match="before capturing"):
        t._rotary_inputs(11, "cpu")
    seen = []
    for capturing in (False, True, True, False):
        t.set_positions(torch.randn(11, 3))
        monkeypatch.setattr(sit, "_capturing", lambda device: False)
        t._rotary_inputs(11, "cpu")
        monkeypatch.setattr(sit, "_capturing", lambda device, c=capturing: c)
        for _ in range(2):                                       # two layers
            pos, freqs = t._rotary_inputs(11, "cpu")
        seen.append((weakref.ref(freqs), pos.data_ptr(), pos.clone()))
        del pos, freqs
    t.set_positions(torch.randn(11, 3))
    assert [ref() is not None for ref, _, _ in seen] == [False, True, True, False]
    assert len(t._positions_captured) == 2
    for (pos, freqs), (ref, ptr, was) in zip(t._positions_captured, seen[1:3]):
        assert freqs is ref() and pos.data_ptr() == ptr and torch.equal(pos, was)


def test_positions_set_and_first_used_in_inference_mode_train_later(mods):
    sit, _ = mods
    for set_inside in (False, True):
        t = sit.SiT(**KW, rotary=(4, 4, 4)).transformer
        given = torch.randn(11, 3)
        if not set_inside:
            t.set_positions(given)
        with torch.inference_mode():
            if set_inside:
                t.set_positions(given)
            t._rotary_inputs(11, "cpu")
        pos, freqs = t._rotary_inputs(11, "cpu")
        assert not pos.is_inference() and not freqs.is_inference() and torch.equal(pos, given)

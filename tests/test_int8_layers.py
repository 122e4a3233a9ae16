"""Layers that serve in 8 bits (FullyConnectedLayer.quantize_int8_): copies and snapshots, and the way back to fp32."""
import copy
import io
import pickle

import pytest
import torch

from stylegan_v_amd.training.layers import FullyConnectedLayer, MappingNetwork


def _layer():
    torch.manual_seed(0)
    return FullyConnectedLayer(64, 48, activation='lrelu', lr_multiplier=0.01)


def _pickled(layer):
    return pickle.loads(pickle.dumps(layer))


def _saved(layer):
    buf = io.BytesIO()
    torch.save(layer, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)           # (what this test wrote)


@pytest.mark.parametrize('copied', [copy.deepcopy, copy.copy, _pickled, _saved])
def test_a_copy_holds_no_derived_rows_and_does_not_serve(copied, monkeypatch):
    layer, x = _layer(), torch.randn([5, 64])
    plain = len(pickle.dumps(layer))
    with torch.no_grad():
        want = layer(x)
        served = layer.quantize_int8_()(x)
        assert len(pickle.dumps(layer)) < plain + 256         # a snapshot is no larger
        # another process: counters start again, and an allocator may return the addresses of before
        monkeypatch.setattr(FullyConnectedLayer, '_parameter_state', lambda self: ((torch.device('cpu'), torch.float32, 64, 0),))
        layer.quantize_int8_()
        layer.weight.data.mul_(2.0)                           # (rows that are stale in a way no counter shows)
        twin = copied(layer)
        assert not any(isinstance(t, torch.Tensor) for t in twin._int8)
        with pytest.raises(RuntimeError, match='quantise it again'):
            twin(x)
        monkeypatch.undo()
        assert torch.equal(twin.quantize_int8_()(x), _requantised(twin)(x)) and not torch.equal(twin(x), served)
    assert torch.equal(twin(x).detach(), _fp32(twin)(x)) and not torch.equal(twin(x), want)      # gradients enabled: the fp32 layer
    assert layer._int8[0] is not None                         # the original keeps its rows


def _fp32(layer):
    fresh = _layer()
    fresh.load_state_dict(layer.state_dict())
    return fresh


def _requantised(layer):
    return _fp32(layer).quantize_int8_()


def test_a_snapshot_from_before_the_rule_does_not_serve(monkeypatch):
    """A pickle that holds the rows beside the parameters, as it was written once."""
    layer, x = _layer(), torch.randn([5, 64])
    layer.quantize_int8_()
    old = _layer()
    state = dict(layer.__dict__)
    state['_int8'] = layer._int8
    monkeypatch.setattr(FullyConnectedLayer, '_parameter_state', lambda self: layer._int8[3])
    old.__setstate__(state)
    with torch.no_grad(), pytest.raises(RuntimeError, match='quantise it again'):
        old(x)


def test_layers_that_never_served_copy_as_before():
    layer, x = _layer(), torch.randn([5, 64])
    for twin in (copy.deepcopy(layer), _pickled(layer)):
        assert twin._int8 is None and '_int8' not in twin.__dict__
        with torch.no_grad():
            assert torch.equal(twin(x), layer(x))


def test_the_way_back_to_fp32():
    layer, x = _layer(), torch.randn([5, 64])
    with torch.no_grad():
        want = layer(x)
        assert not torch.equal(layer.quantize_int8_()(x), want)
        assert layer.drop_int8_() is layer and torch.equal(layer(x), want) and not layer.serves_int8()
        layer.quantize_int8_().weight.add_(0.5)              # one that would refuse
        assert torch.equal(layer.drop_int8_()(x), _fp32(layer)(x))
        twin = copy.deepcopy(layer.quantize_int8_())
        assert torch.equal(twin.drop_int8_()(x), _fp32(layer)(x))
        net = MappingNetwork(z_dim=32, c_dim=3, w_dim=32, num_ws=4, num_layers=2).eval()
        z, c = torch.randn([16, 32]), torch.randn([16, 3])
        want = net(z, c)
        assert not torch.equal(net.quantize_int8_()(z, c), want)
        assert net.drop_int8_() is net and torch.equal(net(z, c), want)


def test_a_network_is_quantised_whole_or_not_at_all():
    net = MappingNetwork(z_dim=32, c_dim=3, w_dim=32, num_ws=4, num_layers=2, activation='tanh').eval()      # (its embedding is linear)
    z, c = torch.randn([16, 32]), torch.randn([16, 3])
    with torch.no_grad():
        want = net(z, c)
        with pytest.raises(RuntimeError, match='tanh'):
            net.quantize_int8_()
        assert torch.equal(net(z, c), want) and net.embed._int8 is None

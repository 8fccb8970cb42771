"""nn.GatedDelta: the operators of a sequence layer together, token by token, over whole
sequences, in training and in 8 bits."""
import pytest
import torch

import brainstate_amd as bs

pytestmark = pytest.mark.gpu


def _layer(dtype=torch.float32, d=96, **kw):
    return bs.nn.GatedDelta(d, 4, 24, num_key_heads=2, key_size=16, dtype=dtype, seed=3, **kw)


def _input(b, t, d=96, dtype=torch.float32):
    rng = torch.Generator().manual_seed(5)
    x = torch.randn(b, t, d, generator=rng).to('cuda', dtype)
    return x, bs.ops.norm_gate_residual(x, torch.ones(d, device='cuda'))[0]


@pytest.mark.parametrize('t', [1, 63, 130])
def test_tokens_one_by_one_give_what_the_sequence_gives(t):
    # both in 32 bits, apart only by the order of sums: some 1e-6 a stage, norms and recurrence
    # enlarge it by a few tens
    layer = _layer()
    stream, normed = _input(3, t)
    layer.init_state(3)
    n_all, s_all = layer(normed, stream)
    last = layer.S.value
    layer.init_state(3)
    for i in range(t):
        n, s = layer(normed[:, i], stream[:, i])
        assert (n - n_all[:, i]).abs().max() < 1e-4
        assert (s - s_all[:, i]).abs().max() < 1e-4
    assert (layer.S.value - last).abs().max() < 1e-4


def test_a_sequence_goes_on_from_the_last_states():
    layer = _layer()
    stream, normed = _input(2, 150)
    layer.init_state(2)
    n_all, _ = layer(normed, stream)
    layer.init_state(2)
    parts = [layer(normed[:, a:b], stream[:, a:b])[0] for a, b in ((0, 70), (70, 71), (71, 150))]
    assert (torch.cat(parts, 1) - n_all).abs().max() < 1e-4


def test_gradients_reach_every_parameter():
    layer = _layer()
    stream, normed = _input(2, 70)
    names = ['weight_in', 'weight_out', 'head_norm', 'next_norm', 'scale', 'log_decay',
             'decay_bias']
    states = {n: getattr(layer, n) for n in names}

    def loss():
        layer.init_state(2)
        n, s = layer(normed, stream)
        return (n * n.roll(1, -1)).mean() + (s * s).mean()

    grads = bs.transform.grad(loss, states)()
    for n in names:
        # a step along the gradient changes the loss by |gradient|^2 times its length: seen in
        # 32 bits to 2%, with a step that changes the loss by 1e-3 (rounding 1e-7 / 1e-3, the
        # second difference cancels in the central one)
        w, g = states[n].value, grads[n]
        norm2 = g.double().square().sum().item()
        assert norm2 > 0
        step = 1e-3 / norm2
        step = min(step, 0.02 * w.norm().item() / norm2 ** 0.5)
        got = []
        for sign in (1, -1):
            states[n].value = w.detach() + sign * step * g
            with torch.no_grad():
                got.append(loss().double().item())
        states[n].value = w
        assert abs((got[0] - got[1]) / (2 * step * norm2) - 1) < 0.02, n


def test_8_bit_projections_stay_near():
    # rows of normal values have a largest of some 4 sigma: rounding to steps of 4/127 leaves
    # 0.9% of sigma on both operands, 1.3% a projection; decay, gate and two norms follow
    layer = _layer(torch.bfloat16, d=512)
    stream, normed = _input(4, 65, 512, torch.bfloat16)
    layer.init_state(4)
    want, _ = layer(normed, stream)
    layer.quantize()
    layer.init_state(4)
    with torch.no_grad():
        got, _ = layer(normed, stream)
        err = (got.float() - want.float()).square().mean().sqrt()
        assert err < 0.1 * want.float().square().mean().sqrt()
        layer.init_state(4)
        for i in range(65):
            n, _ = layer(normed[:, i], stream[:, i])
            err = (n.float() - want[:, i].float()).square().mean().sqrt()
            assert err < 0.1 * want[:, i].float().square().mean().sqrt()


def test_refusals():
    with pytest.raises(ValueError, match='heads'):
        bs.nn.GatedDelta(8, 4, 8, num_key_heads=3)
    with pytest.raises(ValueError, match='outside'):
        bs.nn.GatedDelta(8, 4, 129)
    layer = _layer()
    layer.init_state(2)
    x = torch.zeros(2, 95, device='cuda')
    with pytest.raises(ValueError, match='normed and stream'):
        layer(x, x)
    x = torch.zeros(3, 96, device='cuda')
    with torch.no_grad(), pytest.raises(ValueError, match='states'):
        layer(x, x)

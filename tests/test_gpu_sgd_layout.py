"""FlatSGD and weights in channels-last order: the layout that models.AlphaZero(norm='group') gives its weights, so that no
convolution copies them, and that a batch-normalised network may have been given."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu
LAST = torch.channels_last


def test_channels_last_weights_keep_their_layout():
    from alphazero_amd.optim import FlatSGD
    conv = torch.nn.Conv2d(8, 16, 3).cuda().to(memory_format=LAST)
    w = conv.weight.detach().clone(memory_format=torch.preserve_format)
    opt = FlatSGD(conv.parameters(), lr=0.1, momentum=0.9, weight_decay=1e-2)
    assert conv.weight.is_contiguous(memory_format=LAST) and torch.equal(conv.weight, w)
    assert conv.weight.grad.stride() == conv.weight.stride() == w.stride() and not conv.weight.grad.any()
    ref = torch.nn.Parameter(w.clone(memory_format=torch.preserve_format))
    plain = torch.optim.SGD([ref], lr=0.1, momentum=0.9, weight_decay=1e-2)
    for k in range(3):
        opt.zero_grad()
        conv(torch.randn(2, 8, 6, 7, device='cuda')).square().sum().backward()
        ref.grad = conv.weight.grad.clone(memory_format=torch.preserve_format)
        opt.step()
        plain.step()
        # (three steps of some ten roundings each, of values and updates of this size)
        assert torch.allclose(conv.weight, ref, rtol=1e-6, atol=30 * 2.0 ** -24 * float(ref.grad.abs().max()))


@pytest.mark.parametrize('channels,groups', [(32, None), (24, 2), (20, 5)])
def test_group_normalised_network_with_sgd(channels, groups):
    """Six steps beside torch.optim.SGD, each from the same weights on the same batch.  FlatSGD packs its tensors without
    gaps: the norms' weights lie off 16-byte borders here.  Tolerance of an update: lr (1 + momentum + ...) times what two
    float32 evaluations of a gradient are apart, some 2^-24 for each of the at most 20 000 terms that are added."""
    from alphazero_amd.models import AlphaZeroC4
    from alphazero_amd.optim import FlatSGD
    nets = []
    for _ in range(2):
        torch.manual_seed(4)
        nets.append(AlphaZeroC4(2, channels, norm='group', norm_groups=groups).cuda())
    a, b = nets
    strides = [p.stride() for p in b.parameters()]
    oa = torch.optim.SGD(a.parameters(), lr=0.05, momentum=0.9, weight_decay=1e-4)
    ob = FlatSGD(b.parameters(), lr=0.05, momentum=0.9, weight_decay=1e-4)
    for name in ('_c1', '_c2'):
        w = getattr(b._tower[0], name).weight
        assert w.is_contiguous(memory_format=LAST) and w.grad.is_contiguous(memory_format=LAST)
    g = torch.Generator().manual_seed(1)
    for step in range(6):
        x = (torch.rand(32, 2, 6, 7, generator=g) < 0.3).float().cuda()
        valid = torch.ones(32, 7, dtype=torch.bool, device='cuda')
        with torch.no_grad():
            for p, q in zip(a.parameters(), b.parameters()):
                q.copy_(p)
        outs = []
        for m, o in ((a, oa), (b, ob)):
            o.zero_grad()
            p_hat, v_hat = m(x, valid)
            (p_hat.square().mean() + v_hat.square().mean()).backward()
            outs.append((p_hat.detach(), v_hat.detach()))
        assert all(torch.allclose(s, t, rtol=1e-4, atol=1e-5) for s, t in zip(*outs))
        for p, q in zip(a.parameters(), b.parameters()):
            assert torch.allclose(p.grad, q.grad, rtol=1e-3, atol=20000 * 2.0 ** -24 * float(p.grad.abs().max())), step
        oa.step()
        ob.step()
        for p, q in zip(a.parameters(), b.parameters()):
            assert torch.allclose(p, q, rtol=1e-6, atol=0.5 * 20000 * 2.0 ** -24 * float(p.grad.abs().max())), step
    assert [p.stride() for p in b.parameters() if p.dim() != 4 or p.shape[2] > 1] == [
        s for p, s in zip(b.parameters(), strides) if p.dim() != 4 or p.shape[2] > 1]


def test_a_channels_last_batch_normalised_network_keeps_the_handwritten_pass():
    """The hand-written training pass reads its weights in the plain order; a network in the other one is brought to it."""
    from alphazero_amd.loss import AlphaZeroLoss
    from alphazero_amd.models import AlphaZeroC4
    from alphazero_amd.training import TrainingWorker
    hands = []
    for layout in (torch.contiguous_format, LAST):
        for kind in ('sgd', 'adamw'):
            torch.manual_seed(3)
            net = AlphaZeroC4(1, 32).to(memory_format=layout)
            config = types.SimpleNamespace(Model=lambda: net, Loss=AlphaZeroLoss, training=dict(
                batch_size=16, lr=0.1, momentum=0.9, weight_decay=1e-4, lr_schedule=[5], lr_schedule_gamma=0.1, optimizer=kind))
            tw = TrainingWorker(config, None, [], None, 'cuda')
            assert tw._hand is not None
            g = torch.Generator().manual_seed(2)
            x = (torch.rand(16, 2, 6, 7, generator=g) < 0.3).float().cuda()
            tw._hand.run(x, torch.full((16, 7), 1 / 7, device='cuda'), torch.zeros(16, device='cuda'), torch.ones(16, 7, dtype=torch.bool, device='cuda'))
            hands.append([p.grad.clone() for p in tw.model.parameters()])
    for other in hands[1:]:
        assert all(torch.equal(s, t) for s, t in zip(hands[0], other))

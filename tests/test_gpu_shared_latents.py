"""The table lookup, its gradient and the optimizer as a training step uses them: Gaussians that share their neural
latents through a codebook, rendered, with a loss, and FusedAdamW over the codebook and all other parameters."""
import numpy as np
import pytest
import torch

import synthetic as S
from fgs_testutil import settings_for
from oracle import adamw as O

pytestmark = pytest.mark.gpu

N, ENTRIES, FEATURES = 20_000, 300, 32


def _scene(cuda):
    import FasterGSVDACudaBackend as F
    F.initialize_appearance('neural', 0, 'none', 'tanh', 'relu', True)
    F.initialize_residual_mlp(80, 3, {'otype': 'Identity'}, {'otype': 'FullyFusedMLP', 'activation': 'ReLU', 'output_activation': 'None',
                                                             'n_neurons': 64, 'n_hidden_layers': 2}, False, 1, [0, 1, 2, 3])
    geo = S.geometry(N)
    geo['scales'] = geo['scales'] + 1.0
    prims = {**geo, **S.neural_appearance(N, feature_dim=FEATURES, layer_shapes=S.mlp_layer_shapes(80, 64, 2))}
    r = torch.Generator().manual_seed(5)
    codebook = prims.pop('residual_params').reshape(N, FEATURES)[:ENTRIES].clone()
    leaves = {k: torch.nn.Parameter(v.to(cuda).contiguous()) for k, v in prims.items()}
    leaves['codebook'] = torch.nn.Parameter(codebook.to(cuda).contiguous())
    codes = torch.randint(0, ENTRIES - 7, (N,), generator=r).to(cuda)  # some entries belong to no Gaussian
    settings = settings_for(F, S.ring_cameras(3, 160, 120)[1], 3, cuda)
    target = torch.rand(3, 120, 160, generator=r).to(cuda)
    return F, leaves, codes, settings, target


def _render(F, p, latents, settings):
    return F.diff_rasterize(p['means'], p['scales'], p['rotations'], p['opacities'], torch.empty(0, device=latents.device), settings,
                            base_colors=p['base_colors'], residual_params=latents, mlp_weights=p['mlp_weights'])


@pytest.mark.parametrize('bits', [32, 8])
def test_training_steps_with_a_codebook(cuda, bits):
    from trainer import FusedLoss
    F, p, codes, settings, target = _scene(cuda)
    loss_fn = FusedLoss()
    lrs = {'means': 1e-4, 'scales': 5e-3, 'rotations': 1e-3, 'opacities': 5e-2, 'base_colors': 2.5e-3, 'codebook': 2e-3, 'mlp_weights': 3e-3}
    opt = F.FusedAdamW([{'params': [p[k]], 'lr': lr} for k, lr in lrs.items()], eps=1e-15, weight_decay=0.0, state_bits=bits, max_grad_norm=1e-3)
    for step in range(1, 4):
        opt.zero_grad(set_to_none=True)
        latents = F.embedding_lookup(p['codebook'], codes)
        latents.retain_grad()
        image = _render(F, p, latents, settings)
        _, grad_image = loss_fn(image.detach(), target)
        image.backward(grad_image)
        # the codebook's gradient is the sum of the latents' gradients (here in 64 bits) by entry
        g = latents.grad.double().cpu().numpy()
        want, size, count = np.zeros((ENTRIES, FEATURES)), np.zeros((ENTRIES, FEATURES)), np.zeros(ENTRIES)
        np.add.at(want, codes.cpu().numpy(), g)
        np.add.at(size, codes.cpu().numpy(), np.abs(g))
        np.add.at(count, codes.cpu().numpy(), 1)
        got = p['codebook'].grad.double().cpu().numpy()
        assert (np.abs(got - want) <= 2.0 ** -24 * (count[:, None] * size + 3 * np.abs(want)) + 2.0 ** -149).all()
        assert want.any() and not got[ENTRIES - 7:].any()
        m, v = opt.read_moments()
        before = [(q.detach().cpu().numpy().reshape(-1), a.cpu().numpy().reshape(-1), b.cpu().numpy().reshape(-1))
                  for q, a, b in zip([p[k] for k in lrs], m, v)]
        opt.step()
        norm = np.sqrt(sum((p[k].grad.double() ** 2).sum().item() for k in lrs))
        assert abs(float(opt.grad_norm) - norm) <= 18 * 2.0 ** -24 * norm
        clip = min(1.0, 1e-3 / (norm + 1e-6))
        for (k, lr), (q, a, b) in zip(lrs.items(), before):
            args = (q, a, b, clip * p[k].grad.double().cpu().numpy().reshape(-1), step, lr, (0.9, 0.999), 1e-15, 0.0)
            w, _, _ = O.step64(*args)
            tol, _, _ = O.bounds(*args, clipped=True)
            assert (np.abs(p[k].detach().cpu().numpy().reshape(-1) - w) <= tol).all(), k
    # entries without a Gaussian: no gradient, and without weight decay no change
    assert all(torch.isfinite(q).all() for q in p.values())


def test_rendering_reads_the_looked_up_latents(cuda):
    """Looked-up latents are the gathered rows bit for bit, so the image is the one of the gathered latents."""
    F, p, codes, settings, _ = _scene(cuda)
    with torch.no_grad():
        latents = F.embedding_lookup(p['codebook'], codes)
        assert torch.equal(latents, p['codebook'][codes])
        image = F.rasterize(p['means'], p['scales'], p['rotations'], p['opacities'], settings, True, False, base_colors=p['base_colors'],
                            residual_params=latents, mlp_weights=p['mlp_weights'])
        again = F.rasterize(p['means'], p['scales'], p['rotations'], p['opacities'], settings, True, False, base_colors=p['base_colors'],
                            residual_params=p['codebook'][codes], mlp_weights=p['mlp_weights'])
    assert torch.equal(image, again)


def test_morton_ordering_gathers_rows(cuda):
    """Trainer.apply_morton_ordering orders its rows with the lookup: the same bits as indexing."""
    from trainer import Trainer, morton_order
    prims = {k: v.to(cuda) for k, v in {**S.geometry(5003), **S.sh_appearance(5003, 3)}.items()}
    lrs = {k: 1e-3 for k in prims}
    t = Trainer(prims, lrs, cuda)
    t.exp_avg.normal_()
    t.exp_avg_sq.uniform_()
    order = morton_order(prims['means'])
    moments = {g.name: (t.shard_view(t.exp_avg, g.name)[:t.n].clone(), t.shard_view(t.exp_avg_sq, g.name)[:t.n].clone()) for g in t.groups}
    t.apply_morton_ordering()
    for g in t.groups:
        assert torch.equal(t.view(t.params, g.name).reshape(t.n, -1), prims[g.name].reshape(t.n, -1)[order])
        assert torch.equal(t.shard_view(t.exp_avg, g.name)[:t.n], moments[g.name][0][order])
        assert torch.equal(t.shard_view(t.exp_avg_sq, g.name)[:t.n], moments[g.name][1][order])


@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_training_step_within_compiled_functions(cuda, backend):
    """torch.compile leaves the lookup, its gradient, the step and the reading of moments out of its graphs: the bits of the
    calls outside."""
    import FasterGSVDACudaBackend as F
    r = torch.Generator().manual_seed(1)
    start = torch.randn(30, 16, generator=r).to(cuda)
    idx = torch.randint(0, 30, (100,), generator=r).to(cuda)
    results = []
    for wrap in (lambda f: f, torch.compile(backend=backend)):
        torch._dynamo.reset()
        table = torch.nn.Parameter(start.clone())
        opt = F.FusedAdamW([table], state_bits=8, max_grad_norm=0.5)

        @wrap
        def loss_of(t, i):
            return (F.embedding_lookup(t * 2.0, i, scale=2.0) + 1.0).square().sum()

        @wrap
        def step():
            opt.step()
            return opt.read_moments()

        for _ in range(2):
            opt.zero_grad()
            loss = loss_of(table, idx)
            loss.backward()
            moments = step()
        results.append([loss.detach(), table.detach(), table.grad, opt.grad_norm, *moments[0], *moments[1]])
    assert all(torch.equal(a, b) for a, b in zip(*results))

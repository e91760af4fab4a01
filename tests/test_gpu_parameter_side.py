"""GPU: the parameter side of a training step as it is used -- rows looked up, a loss, the table's gradient, the norm over all
gradients, clipping inside Adam -- against torch in 64 bits; and the framework's own paths that call it."""
import pytest
import torch

from helpers import load_golden
from neuradar_amd import ops
from neuradar_amd.encodings import Embedding
from neuradar_amd.step import FlatAdam

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def torch_adam64(params, grads_of, steps, lr, eps, max_norm, wd=0.0):
    """Clipped AdamW in 64 bits: params (list of tensors) after `steps` steps of gradients grads_of(params, k), and the norms."""
    ps = [p.detach().double().cpu().requires_grad_(True) for p in params]
    opt = torch.optim.AdamW(ps, lr=lr, eps=eps, weight_decay=wd)
    norms = []
    for k in range(steps):
        for p, g in zip(ps, grads_of(ps, k)):
            p.grad = g
        norms.append(float(torch.nn.utils.clip_grad_norm_(ps, max_norm)))
        opt.step()
    return ps, norms


@pytest.mark.parametrize("direct", [False, True])
def test_training_run(direct):
    """Ten clipped steps on a table and a linear layer.  eps is of the gradients' size, so that Adam does not divide the clip factor
    out again.  Tolerance: a step's update is smooth in its gradient, whose fp32 error is 2^-24 times the additions of the longest
    sum (a few hundred) of sums that cancel by less than 100: 1e-3 of an update, ten updates of at most lr."""
    torch.manual_seed(0)
    rows, dim, n, steps, lr, eps = 500, 24, 6000, 10, 1e-2, 0.05
    emb = Embedding(rows, dim, scale=2.0, padding_idx=0).to(DEV)
    head = torch.nn.Linear(dim, 8).to(DEV)
    idx = ((rows + 1.0) ** torch.rand(steps, n, dtype=torch.float64) - 1).long().clamp(0, rows - 1)
    target = torch.randn(steps, n, 8)
    params = [emb.embedding.weight, head.weight, head.bias]

    def grads64(ps, k):
        x = torch.nn.functional.embedding(idx[k], ps[0], padding_idx=0) * 2.0
        loss = ((torch.nn.functional.linear(x, ps[1], ps[2]) - target[k].double()) ** 2).sum(-1).mean()
        return torch.autograd.grad(loss, ps)

    want, norms = torch_adam64(params, grads64, steps, lr, eps, 0.5)
    assert min(norms) > 0.5  # every step is clipped
    opt = FlatAdam(params, lr=lr, eps=eps, warmup_steps=0, max_norm=0.5)
    for k in range(steps):
        loss = ((head(emb(idx[k].to(DEV))) - target[k].to(DEV)) ** 2).sum(-1).mean()
        if direct:
            with ops.direct_param_grads():
                loss.backward()
        else:
            loss.backward()
        opt.step()
        assert abs(float(opt.total_norm) - norms[k]) <= 1e-4 * norms[k]
    for p, w in zip(params, want):
        assert float((p.detach().double().cpu() - w.detach()).abs().max()) <= 1e-3 * steps * lr
    assert not bool(emb.embedding.weight[0].any())


def test_flat_adam_clips_like_torch():
    torch.manual_seed(1)
    shapes = ((64, 32), (64,), (1 << 17, 2), (3,))
    params = [torch.nn.Parameter(torch.randn(*s, device=DEV)) for s in shapes]
    gs = [[torch.randn(*s) * 0.01 for s in shapes] for _ in range(4)]
    opt = FlatAdam(params, lr=1e-2, eps=0.01, weight_decay=1e-3, adamw=True, warmup_steps=0, max_norm=1.0)
    want, norms = torch_adam64(params, lambda ps, k: [g.double() * (1.0 if k != 2 else 0.01) for g in gs[k]], 4, 1e-2, 0.01, 1.0, 1e-3)
    assert norms[0] > 1.0 > norms[2]  # clipped, and not
    for k in range(4):
        for p, g in zip(params, gs[k]):
            p.grad.copy_(g * (1.0 if k != 2 else 0.01))
        opt.step()
        assert abs(float(opt.total_norm) - norms[k]) <= 1e-6 * norms[k]
        assert all(not bool(p.grad.any()) for p in params)
    for p, w in zip(params, want):  # (one fp32 Adam step is off by a few 2^-24 of the parameter and of the update)
        assert float((p.detach().double().cpu() - w.detach()).abs().max()) <= 4 * (8 * 2.0 ** -24 * float(w.detach().abs().max()) + 1e-5 * 1e-2)


def test_clipped_step_replays_as_a_graph():
    torch.manual_seed(2)

    def make():
        torch.manual_seed(3)
        ps = [torch.nn.Parameter(torch.randn(5000, device=DEV)), torch.nn.Parameter(torch.randn(1 << 17, device=DEV))]
        return ps, FlatAdam(ps, lr=1e-2, eps=0.01, warmup_steps=0, max_norm=0.7)

    (pa, oa), (pb, ob) = make(), make()
    static = [torch.zeros_like(p) for p in pb]

    def step_b():
        for p, g in zip(pb, static):
            p.grad.copy_(g)
        ob.step()

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step_b()
    for k in range(4):
        gs = [torch.randn_like(p) * (0.001 if k == 2 else 1.0) for p in pa]
        for p, g, s in zip(pa, gs, static):
            p.grad.copy_(g)
            s.copy_(g)
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(oa.total_norm, ob.total_norm)
        for p, q in zip(pa, pb):
            assert torch.equal(p.detach(), q.detach())


def test_fused_step_clips_every_group():
    """FusedTrainStep with a max_norm on the tables: one step's first moments are (1 - beta1) times the clipped gradients of the
    modular path (whose agreement with the fused step is 1e-3 of a tensor's largest gradient)."""
    from neuradar_amd.fused_step import FusedTrainStep
    from neuradar_amd.rays import RayBundle
    from test_gpu_parity import build_hot_path, dev

    g = load_golden("pipeline")
    o, d, area, fars = dev(g["origins"]), dev(g["directions"]), dev(g["pixel_area"]), dev(g["fars"])
    t_rand, j1, j2 = dev(g["t_rand"]), dev(g["jitter1"]), dev(g["jitter2"])
    tf, td = dev(g["target_features"]), dev(g["target_depth"])
    ref = build_hot_path(g).train()
    ref.bench_loss(ref.get_nff_outputs(RayBundle(o, d, area, fars=fars.clone()), t_rand=t_rand, jitters=(j1, j2)), tf, td).backward()
    model = build_hot_path(g).train()
    groups, skip = model.get_param_groups(), list(model.proposal_fields[0].parameters())
    tables = [p for p in ref.get_param_groups()["hashgrids"] if p.grad is not None and bool(p.grad.any())]
    norm = float(torch.stack([p.grad.double().square().sum() for p in tables]).sum().sqrt())
    opts = [FlatAdam(groups["hashgrids"], lr=1e-2, warmup_steps=0, skip=skip, max_norm=0.25 * norm),
            FlatAdam(groups["fields"], lr=1e-2, warmup_steps=0, skip=skip)]
    fused = FusedTrainStep(model, o.shape[0])
    fused.forward_backward(o, d, area[:, 0].contiguous(), fars[:, 0].contiguous(), tf, td[:, 0].contiguous(), t_rand,
                           j1[:, 0].contiguous(), j2[:, 0].contiguous(), optimizers=opts)
    assert abs(float(opts[0].total_norm) - norm) <= 2e-3 * norm
    names = {n: p for n, p in ref.named_parameters()}
    checked = 0
    for n, p in model.named_parameters():
        for opt, factor in ((opts[0], 0.25), (opts[1], 1.0)):
            try:
                i = opt.buffer_of(p)
            except KeyError:
                continue
            want = names[n].grad
            if want is None or any(p is s for s in skip):
                continue
            at = (p.data_ptr() - opt.buffers[i][0].data_ptr()) // 4
            m = opt.state[i][0].reshape(-1)[at:at + p.numel()]
            assert not bool(opt.buffers[i][1].any())
            err = (m - 0.1 * factor * want.reshape(-1)).abs().max()
            assert float(err) <= 0.1 * factor * 2e-3 * float(want.abs().max()) + 1e-12, (n, float(err))
            checked += 1
    assert checked > 5
    with pytest.raises(NotImplementedError, match="reducer"):
        fused.forward_backward(o, d, area[:, 0].contiguous(), fars[:, 0].contiguous(), tf, td[:, 0].contiguous(), t_rand,
                               j1[:, 0].contiguous(), j2[:, 0].contiguous(), optimizers=opts, reducer=object())


def test_model_appearance_rows_with_sorted_gradient():
    from neuradar_amd.step import HotPathConfig, NeuRadarHotPath

    torch.manual_seed(4)
    outs, grads = [], []
    times, sensor = torch.rand(3000, device=DEV) * 20.0, torch.randint(0, 3, (3000,), device=DEV)
    w = torch.randn(3000, 16, device=DEV)
    for flag in (False, True):
        torch.manual_seed(5)
        cfg = HotPathConfig(appearance_dim=16, num_sensors=3, sorted_appearance_grad=flag)
        cfg.field.grid.static.log2_hashmap_size = cfg.proposal_field_1.grid.static.log2_hashmap_size = 12
        cfg.proposal_field_2.grid.static.log2_hashmap_size = 12
        model = NeuRadarHotPath(cfg).to(DEV).train()
        out = model.appearance_of(times, sensor)
        (out * w).sum().backward()
        outs.append(out.detach())
        grads.append(model.appearance_embedding.weight.grad.double())
    assert torch.equal(*outs)
    # both sum about 100 products of size |w| <= 5 in fp32
    assert float((grads[0] - grads[1]).abs().max()) <= 200 * 2.0 ** -24 * 500

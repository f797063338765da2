"""The training step with group norm in the encoder (GraphVAE(norm="group")), activations kept in 32 or in
8 bits, against a float64 restatement on the CPU.

Tolerances: values and gradients pass through fp32 kernels whose worst amplification is the norm's
1 / sqrt(var + eps) <= 316 of a rounding 2^-24; ten roundings on the way to it make 1.9e-4 of a tensor's
largest entry: 2e-4.  With 8-bit checkpoints the reference quantises its own activations; where one lies
within rounding of the middle between two codes the kernels may take the other code, which moves one of
at least a thousand summands by 1/64: 32 such values would make 5e-4, so 1e-3 together."""
import sys
from pathlib import Path

import numpy as np
import pytest
import torch
import torch.nn.functional as F

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT)); sys.path.insert(0, str(ROOT / "graph-vae_amd"))
from oracle import ref_step as ref  # noqa: E402
from test_norm8 import quantise_ref  # noqa: E402

gpu = pytest.mark.gpu
DEV = "cuda:0"


# ------------------------------------------------------------------ float64 restatement
def _q(t):
    return torch.from_numpy(quantise_ref(t.detach().float().numpy().astype(np.float64))[2])


class _Norm(torch.autograd.Function):
    """Group norm + ReLU of one graph's rows, the backward from the kept input (quantised if asked)."""

    @staticmethod
    def forward(ctx, x, w, b, G, bits):
        n, C = x.shape
        v = x.view(n, G, -1)
        mean = v.mean((0, 2), keepdim=True)
        rstd = (v.var((0, 2), unbiased=False, keepdim=True) + 1e-5).rsqrt()
        y = F.relu(((v - mean) * rstd).view(n, C) * w + b)
        ctx.save_for_backward(_q(x) if bits == 8 else x, w, b, mean, rstd)
        ctx.G = G
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, b, mean, rstd = ctx.saved_tensors
        n, C = x.shape
        h = ((x.view(n, ctx.G, -1) - mean) * rstd)
        dz = dy * ((h.view(n, C) * w + b) > 0)
        g = (dz * w).view_as(h)
        dx = rstd * (g - g.mean((0, 2), keepdim=True) - h * (g * h).mean((0, 2), keepdim=True))
        return dx.view(n, C), (dz * h.view(n, C)).sum(0), dz.sum(0), None, None


class _Linear(torch.autograd.Function):
    """x W^T, the weight gradient from the kept input (quantised if asked)."""

    @staticmethod
    def forward(ctx, x, W, bits):
        ctx.save_for_backward(_q(x) if bits == 8 else x, W)
        return x @ W.t()

    @staticmethod
    def backward(ctx, dy):
        x, W = ctx.saved_tensors
        return dy @ W, dy.t() @ x, None


def reference(state, hb, eps, G, bits):
    """rec, kl and all parameter gradients in float64.  The losses gather prediction and truth through one
    permutation, so the identity serves (rounding of the sum's order aside)."""
    st = {k: v.double() for k, v in ref.make_trainable(state).items()}
    leaves = {k: v.detach().requires_grad_() for k, v in st.items() if k in ref.PARAM_NAMES}
    p = {**st, **leaves}
    recs, kls = [], []
    for g, e in zip(ref.graphs_from_arrays(hb.x, hb.adj_dense, hb.n_x, hb.num_real_nodes), eps.double()):
        N, R = g.adj_dense.size(0), g.num_real_nodes
        A, n = g.adj_dense.double(), g.x.size(0)
        M = torch.zeros(n, n, dtype=torch.float64)
        r = min(R, n)
        M[:r, :r] = (A[:r, :r] != 0).double()
        M.fill_diagonal_(1.0)
        dinv = M.sum(1).pow(-0.5)
        Ahat = dinv[:, None] * M * dinv[None]
        h = _Norm.apply(Ahat @ (g.x.double() @ p["conv1.lin.weight"].t()) + p["conv1.bias"], p["bn1.weight"],
                        p["bn1.bias"], G, bits)
        h = _Norm.apply(Ahat @ _Linear.apply(h, p["conv2.lin.weight"], bits) + p["conv2.bias"], p["bn2.weight"],
                        p["bn2.bias"], G, bits)
        v = h.sum(0) / R
        mu = p["mu.weight"] @ v + p["mu.bias"]
        lv = (p["logvar.weight"] @ v + p["logvar.bias"]).clamp(-4.0, 4.0)
        z = mu + e * torch.exp(0.5 * lv)
        vec = p["dec_edge.2.weight"] @ F.relu(p["dec_edge.0.weight"] @ z + p["dec_edge.0.bias"]) + p["dec_edge.2.bias"]
        node = p["dec_node.2.weight"] @ F.relu(p["dec_node.0.weight"] @ z + p["dec_node.0.bias"]) + p["dec_node.2.bias"]
        tri = torch.triu_indices(R, R, offset=1)
        pred = ref.vec_to_adj(vec, N)
        edges = F.binary_cross_entropy_with_logits(pred[tri[0], tri[1]], A[tri[0], tri[1]],
                                                   pos_weight=p["pos_weight_global"].double())
        truth = torch.zeros(N, dtype=torch.float64)
        truth[:R] = 1.0
        wn = torch.tensor((N - R) / (R + 1e-8), dtype=torch.float64).clamp(1.0, 5.0)
        recs.append(edges + F.binary_cross_entropy_with_logits(node, truth, pos_weight=wn))
        kls.append(-0.5 * torch.mean(1 + lv - mu.pow(2) - lv.exp()))
    rec, kl = torch.stack(recs).mean(), torch.stack(kls).mean()
    (rec + kl).backward()
    return rec.item(), kl.item(), {k: v.grad for k, v in leaves.items()}


def _model(F_, H, Z, N, G, bits, hb, matching="fused", seed=3):
    from graphvae.models import GraphVAE
    torch.manual_seed(seed)
    model = GraphVAE(F_, H, Z, N, matching=matching, norm="group", norm_groups=G, act_bits=bits)
    with torch.no_grad():
        for m in (model.bn1, model.bn2):
            m.weight.add_(0.2 * torch.randn(H))
            m.bias.add_(0.2 * torch.randn(H))
    model.precompute_dataset_rho([hb])
    state = {k: v.detach().clone() for k, v in model.state_dict().items()}
    return model, state


# ------------------------------------------------------------------ host
def test_norm_option_refusals():
    from graphvae.models import GraphVAE
    for kw in [dict(norm="layer"), dict(act_bits=16), dict(act_bits=8), dict(norm="group", norm_groups=3),
               dict(norm="group", norm_groups=0), dict(norm="group", act_bits=4)]:
        with pytest.raises(ValueError):
            GraphVAE(1, 16, 4, 6, **kw)
    a, b = GraphVAE(1, 16, 4, 6), GraphVAE(1, 16, 4, 6, norm="group", norm_groups=4, act_bits=8)
    assert list(a.state_dict()) == list(b.state_dict())
    b.load_state_dict(a.state_dict(), strict=True)


def test_step_entry_points_refuse():
    import ctypes
    from graphvae import engine
    L = engine._bind()
    d, ok = engine.Dims(1, 16, 4, 6), engine.GnOpts(4, 8, 1e-5)
    assert L.gvae_step_gn_ws_bytes(ctypes.byref(d), ctypes.byref(ok), 5) > 0
    assert L.gvae_step_gn_ws_bytes(ctypes.byref(d), ctypes.byref(ok), 0) == 0
    for bad in [(3, 8, 1e-5), (0, 8, 1e-5), (4, 16, 1e-5), (4, 8, 0.0), (4, 8, float("nan"))]:
        o = engine.GnOpts(*bad)
        assert L.gvae_step_gn_ws_bytes(ctypes.byref(d), ctypes.byref(o), 5) == 0
        assert L.gvae_step_gn_forward_model(ctypes.byref(d), ctypes.byref(o), 16, 16, 16, 16, 16, 5, 16, 16, None) == -1
        assert L.gvae_step_gn_backward(ctypes.byref(d), ctypes.byref(o), 16, 16, 16, 16, 16, 5, 16, 16, 0, 1.0, 1.0,
                                       None, 16, 16, None) == -1
    for n in (0, 65536):
        assert L.gvae_step_gn_forward_model(ctypes.byref(d), ctypes.byref(ok), 16, 16, 16, 16, 16, n, 16, 16, None) == -1
    assert L.gvae_step_gn_forward_model(ctypes.byref(d), ctypes.byref(ok), None, 16, 16, 16, 16, 5, 16, 16, None) == -1
    assert L.gvae_step_gn_backward(ctypes.byref(d), ctypes.byref(ok), 16, 16, 16, 16, 16, 5, 16, 16, 3, 1.0, 1.0, None,
                                   16, 16, None) == -1
    # what 8 bits save: the three kept activations take about a quarter
    big = engine.Dims(1, 128, 64, 128)
    full = L.gvae_step_gn_ws_bytes(ctypes.byref(big), ctypes.byref(engine.GnOpts(8, 32, 1e-5)), 512)
    small = L.gvae_step_gn_ws_bytes(ctypes.byref(big), ctypes.byref(engine.GnOpts(8, 8, 1e-5)), 512)
    assert full - small > 0.7 * 3 * 512 * 128 * 128 * 4


# ------------------------------------------------------------------ the step
@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind,B,N,feature,H,G", [("enzymes", 12, 12, "deg", 32, 4), ("enzymes", 5, 20, "id", 48, 8),
                                                  ("dense", 9, 32, "deg", 128, 8), ("enzymes", 3, 40, "deg", 20, 5)])
def test_step_against_float64(kind, B, N, feature, H, G, bits):
    from graphvae.data import synthetic_batch
    hb = synthetic_batch(kind, B, N, feature, seed=5)
    model, state = _model(hb.x.shape[-1], H, 16, N, G, bits, hb)
    eps = torch.randn(B, 16, generator=torch.Generator().manual_seed(1))
    rec, kl, grads = reference(state, hb, eps, G, bits)
    model = model.to(DEV).train()
    out = model.forward_with_eps(hb.to(DEV), eps.to(DEV))
    (out["rec"] + out["kl"]).backward()
    assert abs(out["rec"].item() - rec) <= 2e-4 * abs(rec) and abs(out["kl"].item() - kl) <= 2e-4 * abs(kl)
    tol = 2e-4 if bits == 32 else 1e-3
    for name, p in model.named_parameters():
        want = grads[name]
        assert (p.grad.cpu().double() - want).abs().max() <= tol * want.abs().max(), name
    # evaluation is the same forward: no statistics of the batch, none kept
    model.eval()
    again = model.forward_with_eps(hb.to(DEV), eps.to(DEV))
    assert again["rec"].item() == out["rec"].item() and again["kl"].item() == out["kl"].item()
    assert torch.equal(model.bn1.running_mean.cpu(), state["bn1.running_mean"])
    assert int(model.bn1.num_batches_tracked) == 0


@gpu
@pytest.mark.parametrize("matching", ["fused", "stream"])
def test_bits_leave_the_forward_alone_and_schedules_agree(matching):
    """act_bits changes gradients only (the forward's sums may be taken in another order: 2e-4 as above, here
    on losses of order one); overlapped and pipelined schedules give the bits of the
    sequential one; parameters stay finite."""
    from graphvae.data import synthetic_batch
    from graphvae.train.train_ddp import TrainStep
    N, B = 24, 40
    host = [synthetic_batch("enzymes", B, N, "deg", seed=s) for s in (3, 4)]
    first = {}
    for bits in (32, 8):
        runs = []
        for overlap, pipeline in ((False, False), (True, False), (True, True)):
            model, _ = _model(1, 64, 32, N, 8, bits, host[0], matching)
            model = model.to(DEV).train()
            step = TrainStep(model, 1e-2, 1e-4, 5.0, overlap_matching=overlap, pipeline=pipeline)
            gen = torch.Generator().manual_seed(9)
            outs, perms = [], []
            for s in range(5):
                out4 = step(host[s % 2].to(DEV), 0.5, 1.0, eps=torch.randn(B, 32, generator=gen).to(DEV))
                step.wait()
                outs.append(out4.cpu())
                perms.append(model.last_permutations().cpu())
            model._engine.check_matching()
            runs.append((torch.stack(outs), torch.stack(perms), step.pop_loss_sum().cpu(),
                         model.flat_parameters().detach().cpu().clone()))
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
        assert torch.isfinite(runs[0][3]).all() and int(model.bn2.num_batches_tracked) == 0
        first[bits] = runs[0][0][0]
    assert ((first[32] - first[8]).abs() <= 2e-4 * first[32].abs()).all()     # before any update


@gpu
def test_other_losses_and_growing_batches():
    """forward_old and forward_individual_rho run on the same encoder, gradients are finite, a larger
    batch after a smaller one regrows the workspace, and gradients repeat bit for bit."""
    from graphvae.data import synthetic_batch
    small, large = (synthetic_batch("enzymes", b, 16, "deg", seed=b) for b in (3, 30))
    model, _ = _model(1, 32, 8, 16, 4, 8, large)
    model = model.to(DEV).train()
    for hb in (small, large, small):
        batch = hb.to(DEV)
        for kw in ({}, {"legacy": True}, {"individual_rho": True}):
            eps = torch.randn(batch.num_graphs, 8, generator=torch.Generator().manual_seed(2)).to(DEV)
            got = []
            for _ in range(2):
                model.zero_grad(set_to_none=True)
                out = model.forward_with_eps(batch, eps, **kw)
                (out["rec"] + out["kl"]).backward()
                got.append(torch.cat([p.grad.reshape(-1) for p in model.parameters() if p.grad is not None]))
            assert torch.isfinite(got[0]).all() and torch.equal(got[0], got[1])
    with pytest.raises(Exception, match="not kept"):
        model._engine.debug_tensor("H1", 3)
    assert model._engine.debug_tensor("gvec", 3).shape == (3, 32)


@gpu
@pytest.mark.parametrize("bits", ["8", "32"])
def test_trainer_cli_with_group_norm(tmp_path, capfd, bits):
    """The trainer's command line with the options: epochs run, options are recorded, the checkpoint
    loads strictly and keeps untouched running statistics."""
    import re
    import yaml
    from graphvae.models import GraphVAE
    from graphvae.train import train_ddp as T
    run = tmp_path / "run"
    T.main(["--dataset", "synthetic-dense", "--feature_type", "deg", "--max_nodes", "16", "--epochs", "2", "--norm",
            "group", "--norm_groups", "4", "--act_bits", bits, "--log_dir", str(run), "--no_wandb"])
    losses = re.findall(r"Ep \d+ \| train ([-\d.einfa+]+) \| val ([-\d.einfa+]+)", capfd.readouterr().out)
    assert len(losses) == 2 and all(np.isfinite(float(v)) for pair in losses for v in pair)
    params = yaml.safe_load((run / "params.yaml").read_text())
    assert (params["norm"], params["norm_groups"], params["act_bits"]) == ("group", 4, int(bits))
    sd = torch.load(run / "graphvae_ddp.pt", weights_only=True)
    model = GraphVAE(params["in_dim"], params["hid_dim"], params["z_dim"], 16, norm="group", norm_groups=4)
    model.load_state_dict(sd, strict=True)
    assert int(sd["bn1.num_batches_tracked"]) == 0 and not sd["bn1.running_mean"].any()


@gpu
def test_single_node_graphs_and_equal_nodes():
    """Graphs of one node, and complete graphs whose nodes are all alike (variance from the channels alone):
    finite losses and gradients."""
    from graphvae.data import collate, graph_from_adjacency
    graphs = [np.zeros((1, 1), np.float32), 1.0 - np.eye(6, dtype=np.float32), np.zeros((1, 1), np.float32)]
    hb = collate([graph_from_adjacency(a, 6, "deg") for a in graphs], 6)
    for bits in (32, 8):
        model, _ = _model(1, 16, 4, 6, 4, bits, hb)
        model = model.to(DEV).train()
        out = model.forward_with_eps(hb.to(DEV), torch.zeros(3, 4, device=DEV))
        nodes = out["kl"]
        nodes.backward()
        g = torch.cat([p.grad.reshape(-1) for p in model.parameters() if p.grad is not None])
        assert torch.isfinite(g).all() and torch.isfinite(out["kl"])


def _host_engine(F_, H, Z, N, **norm):
    """The engine's workspace bookkeeping on host memory (nothing is launched)."""
    from graphvae import engine
    eng = object.__new__(engine.StepEngine)
    eng.gn = engine.norm_options(norm.get("norm", "batch"), norm.get("norm_groups", 8), norm.get("act_bits", 32), H)
    eng.L, eng.dims, eng.N, eng.device = engine._bind(), engine.Dims(F_, H, Z, N), N, torch.device("cpu")
    eng._slots, eng._cur, eng._ws_need = [engine._Slot(eng.device)], 0, {}
    return eng


@pytest.mark.parametrize("N,H,sizes", [(32, 128, (513, 512, 513, 100, 512)), (126, 64, (521, 520)), (8, 256, (513, 512)),
                                       (16, 128, (1025, 1024, 1, 1024))])
def test_workspace_holds_every_batch_size(N, H, sizes):
    """A smaller batch can need more scratch than a larger one before it (its rows are cut into more ranges);
    the workspace always holds what the batch at hand needs."""
    import ctypes
    from graphvae import engine
    for kw in ({}, {"norm": "group"}, {"norm": "group", "act_bits": 8}):
        eng = _host_engine(1, H, 64, N, **kw)
        for B in sizes:
            eng._ensure(B)
            need = (eng.L.gvae_step_ws_bytes(ctypes.byref(eng.dims), B) if eng.gn is None else
                    eng.L.gvae_step_gn_ws_bytes(ctypes.byref(eng.dims), ctypes.byref(eng.gn), B))
            assert eng._ws.numel() >= need > 0, (kw, B)


def _load_model(run, device):
    sys.path.insert(0, str(ROOT / "graph-vae_amd" / "experiments"))
    from sample import load_model
    return load_model(run, device)[0]


@pytest.mark.parametrize("entries,want", [({}, ("batch", 8, 32)), ({"norm": None}, ("batch", 8, 32)),
                                          ({"norm": "batch", "norm_groups": 8, "act_bits": 32}, ("batch", 8, 32)),
                                          ({"norm": "group", "norm_groups": 4, "act_bits": 8}, ("group", 4, 8)),
                                          ({"norm": "group", "norm_groups": 2, "act_bits": 32}, ("group", 2, 32))])
def test_a_run_is_loaded_with_its_norm(tmp_path, entries, want):
    import yaml
    from graphvae.models import GraphVAE
    torch.save(GraphVAE(1, 16, 4, 6).state_dict(), tmp_path / "graphvae_ddp.pt")
    (tmp_path / "params.yaml").write_text(yaml.safe_dump({"hid_dim": 16, "z_dim": 4, **entries}))
    model = _load_model(tmp_path, "cpu")
    assert (model.norm, model.norm_groups, model.act_bits) == want


@gpu
def test_a_trained_run_evaluates_as_it_was_trained(tmp_path):
    """A run of the trainer's command line, loaded for sampling: its forward is that of the trained model."""
    from graphvae.data import synthetic_batch
    from graphvae.models import GraphVAE
    from graphvae.train import train_ddp as T
    T.main(["--dataset", "synthetic-dense", "--feature_type", "deg", "--max_nodes", "16", "--epochs", "1", "--norm",
            "group", "--norm_groups", "4", "--act_bits", "8", "--log_dir", str(tmp_path), "--no_wandb"])
    loaded = _load_model(tmp_path, DEV)
    hid, z = loaded.hid_dim, loaded.z_dim
    built = GraphVAE(1, hid, z, 16, norm="group", norm_groups=4, act_bits=8)
    built.load_state_dict(torch.load(tmp_path / "graphvae_ddp.pt", weights_only=True), strict=True)
    hb = synthetic_batch("dense", 7, 16, "deg", seed=6)
    eps = torch.randn(7, z, generator=torch.Generator().manual_seed(6)).to(DEV)
    outs = []
    for model in (loaded, built.to(DEV).eval()):
        model.precompute_dataset_rho([hb])
        with torch.no_grad():
            outs.append(model.forward_with_eps(hb.to(DEV), eps))
    assert all(torch.equal(outs[0][k], outs[1][k]) for k in ("rec", "kl"))


@gpu
@pytest.mark.parametrize("matching", ["fused", "stream"])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_in_flight_equal_the_sequential_schedule(matching, bits):
    """Eleven pipelined steps over four workspaces, batches of two sizes and their noise on the device beforehand and
    nothing waited for or read until the last: losses, their sum and the parameters bit for bit those of
    steps run one after the other."""
    from graphvae.data import synthetic_batch
    from graphvae.train.train_ddp import TrainStep
    N, steps = 24, 11
    host = [synthetic_batch("enzymes", b, N, "deg", seed=b) for b in (40, 57, 41)]
    order = [host[s % 3] for s in range(steps)]
    gen = torch.Generator().manual_seed(9)
    noise = [torch.randn(hb.num_graphs, 32, generator=gen).to(DEV) for hb in order]
    batches = {id(hb): hb.to(DEV) for hb in host}
    runs = []
    for overlap, pipeline in ((False, False), (True, True)):
        model, _ = _model(1, 64, 32, N, 8, bits, host[0], matching)
        model = model.to(DEV).train()
        step = TrainStep(model, 1e-2, 1e-4, 5.0, overlap_matching=overlap, pipeline=pipeline, slots=4)
        torch.cuda.synchronize()
        outs = [step(batches[id(hb)], 0.5, 1.0, eps=e) for hb, e in zip(order, noise)]
        step.wait()
        runs.append([torch.stack(outs).cpu(), step.pop_loss_sum().cpu(), model.flat_parameters().detach().cpu().clone()])
        model._engine.check_matching()
    assert torch.isfinite(runs[0][2]).all() and all(torch.equal(a, b) for a, b in zip(*runs))


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_smaller_batch_behind_a_larger_one(bits):
    """512 graphs behind 513, whose workspace is smaller: losses and gradients are those of a model that has seen the
    512 alone."""
    from graphvae.data import synthetic_batch
    hb = synthetic_batch("dense", 513, 32, "deg", seed=8)
    large, small = hb.to(DEV), hb.index(range(512)).to(DEV)
    eps = torch.randn(513, 16, generator=torch.Generator().manual_seed(8)).to(DEV)
    runs = []
    for batches in ((small,), (large, small)):
        model, _ = _model(1, 128, 16, 32, 8, bits, hb, matching="none")
        model = model.to(DEV).train()
        for b in batches:
            model.zero_grad(set_to_none=True)
            out = model.forward_with_eps(b, eps[:b.num_graphs].contiguous())
            (out["rec"] + out["kl"]).backward()
        runs.append([out["rec"].detach(), out["kl"].detach(), *(p.grad for p in model.parameters() if p.grad is not None)])
    assert all(torch.equal(a, b) for a, b in zip(*runs))

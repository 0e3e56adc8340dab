"""Training with group norms in the place of batch norms (networks/norm.py) and orthogonalised updates (train.MuonAdam): the
operators together, through the networks and the trainer step."""
import copy
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from conftest import tiny_cfg

gpu = pytest.mark.gpu
DEV = "cuda"


def _mixed(dtype=torch.float32):
    g = torch.Generator().manual_seed(0)
    mats = [nn.Parameter(torch.randn(s, generator=g).to(dtype)) for s in ((4, 6), (3, 2, 3, 3))]
    rest = [nn.Parameter(torch.randn(s, generator=g)) for s in ((5,), (1,))]
    return mats, rest


def test_muon_adam_groups_and_state_dicts():
    from boostmvsnerfs_amd.train import MuonAdam, make_lr_scheduler
    mats, rest = _mixed(torch.bfloat16)
    opt = MuonAdam(mats, rest, lr=0.1, adam_lr=1e-3)
    assert [g["muon"] for g in opt.param_groups] == [True, False]
    sched = make_lr_scheduler(opt, 0.5, 1)
    for p in rest:
        p.grad = torch.ones_like(p)
    opt.step()                                               # (matrices without gradients: nothing to launch)
    sched.step()
    assert [g["lr"] for g in opt.param_groups] == [0.05, 5e-4]
    assert float(opt.state[rest[0]]["step"]) == 1
    opt.state[mats[0]]["momentum_buffer"] = torch.full((4, 6), 1 + 2.0 ** -20)
    saved = copy.deepcopy(opt.state_dict())
    again = MuonAdam(*_mixed(torch.bfloat16), lr=0.3, adam_lr=1e-2)
    again.load_state_dict(saved)
    assert [g["lr"] for g in again.param_groups] == [0.05, 5e-4]
    buf = again.state[again.param_groups[0]["params"][0]]["momentum_buffer"]
    assert buf.dtype == torch.float32 and float(buf[0, 0]) == 1 + 2.0 ** -20     # a bf16 weight's momentum stays fp32
    for p in again.param_groups[1]["params"]:
        p.grad = torch.ones_like(p)
    again.step()                                             # Adam goes on from the loaded state, at the loaded rate
    for p in rest:
        p.grad = torch.ones_like(p)
    opt.step()
    for p, q in zip(rest, again.param_groups[1]["params"]):
        assert float(again.state[q]["step"]) == 2
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(opt.state[p][k], again.state[q][k])
    # Adam alone is GroupedAdam, bit for bit
    from boostmvsnerfs_amd.train import GroupedAdam
    ma, ra = _mixed()
    mb, rb = _mixed()
    a, b = MuonAdam(ma, ra, adam_lr=1e-3), GroupedAdam(rb, lr=1e-3)
    for k in range(3):
        for p, q in zip(ra, rb):
            p.grad = q.grad = torch.full_like(p, 0.1 * (k + 1))
        a.step(), b.step()
    assert all(torch.equal(p, q) for p, q in zip(ra, rb))


def test_muon_adam_refusals():
    from boostmvsnerfs_amd.config import make_cfg, set_cfg
    from boostmvsnerfs_amd.networks.enerf.network import Network
    from boostmvsnerfs_amd.train import GroupedAdam, MuonAdam, make_optimizer
    mats, rest = _mixed()
    with pytest.raises(ValueError, match="2 dimensions"):
        MuonAdam(rest)
    with pytest.raises(ValueError, match="scale"):
        MuonAdam(mats, scale="x")
    with pytest.raises(ValueError, match="among the others"):
        MuonAdam(mats, mats[:1])
    opt = MuonAdam(mats, lr=torch.tensor(0.1))
    mats[0].grad = torch.ones_like(mats[0])
    with pytest.raises(TypeError, match="plain numbers"):
        opt.step()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        MuonAdam(mats).step()
    set_cfg(make_cfg("enerf_eval"))
    net = Network()
    assert type(make_optimizer(net)) is GroupedAdam
    opt = make_optimizer(net, optim="muon", lr=3e-4, muon_lr=0.03)
    assert len(opt.param_groups) == 115 and sum(g["muon"] for g in opt.param_groups) == 40
    assert all(g["lr"] == (0.03 if g["muon"] else 3e-4) for g in opt.param_groups)
    with pytest.raises(ValueError, match="optim"):
        make_optimizer(net, optim="sgd")


def test_groups_added_later_step_as_what_they_say_they_are(monkeypatch):
    from boostmvsnerfs_amd import ops
    from boostmvsnerfs_amd.train import GroupedAdam, MuonAdam
    stepped = []
    monkeypatch.setattr(ops, "muon_step", lambda params, *args: stepped.append((list(params), args[2])))
    mats, rest = _mixed()
    for others in ([], rest[:1]):                            # with and without an Adam group from the start
        opt = MuonAdam(mats[:1], others, lr=0.1, adam_lr=1e-3, adam_eps=1e-6)
        late, twin = torch.nn.Parameter(torch.randn(7)), None
        twin = torch.nn.Parameter(late.detach().clone())
        adam = GroupedAdam([twin], lr=1e-3, eps=1e-6)
        opt.add_param_group({"params": late, "muon": False})
        opt.add_param_group({"params": [mats[1]], "lr": 0.5})
        for p in (*mats, *rest, late, twin):
            p.grad = torch.full_like(p, 0.1)
        for _ in range(2):
            stepped.clear()
            opt.step(), adam.step()
            assert torch.equal(late, twin) and float(opt.state[late]["step"]) == float(adam.state[twin]["step"])
            assert [(len(ps), lr) for ps, lr in stepped] == [(1, 0.1), (1, 0.5)]
            assert stepped[0][0][0] is mats[0] and stepped[1][0][0] is mats[1]
        assert set(opt.param_groups[-2]) == set(adam.param_groups[0]) | {"muon"}
        n = len(opt.param_groups)
        for bad, match in (({"params": [torch.nn.Parameter(torch.zeros(5))]}, "2 dimensions"),
                           ({"params": [torch.nn.Parameter(torch.zeros(5, 5))], "scale": "x"}, "scale"),
                           ({"params": [mats[0]], "muon": False}, "among the others"), ({"params": [late]}, "more than one parameter group"),
                           ({"params": [late], "muon": False}, "more than one parameter group")):
            with pytest.raises(ValueError, match=match):
                opt.add_param_group(bad)
            assert len(opt.param_groups) == n                # refused as a whole
        saved = copy.deepcopy(opt.state_dict())
        opt.load_state_dict(saved)
        opt.step(), adam.step()
        assert torch.equal(late, twin)


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "torch"])
def test_muon_adam_survives_copies(how, monkeypatch):
    import io
    import pickle

    from boostmvsnerfs_amd import ops
    from boostmvsnerfs_amd.train import MuonAdam
    lists = []
    monkeypatch.setattr(ops, "muon_step", lambda *args: lists.append(args))
    mats, rest = _mixed()
    opt = MuonAdam(mats, rest, lr=0.1, adam_lr=1e-3, adam_eps=1e-6, adam_weight_decay=0.1)

    def grads(o):
        for g in o.param_groups:
            for p in g["params"]:
                p.grad = torch.full_like(p, 0.1)
    grads(opt)
    opt.step()
    opt.state[mats[0]]["momentum_buffer"].fill_(0.5)
    if how == "deepcopy":
        twin = copy.deepcopy(opt)
    elif how == "pickle":
        twin = pickle.loads(pickle.dumps(opt))
    else:
        f = io.BytesIO()
        torch.save(opt, f)
        f.seek(0)
        twin = torch.load(f, weights_only=False)             # (this test's own bytes)
    mine, theirs = ([p for g in o.param_groups for p in g["params"]] for o in (opt, twin))
    assert not {id(p) for p in mine} & {id(p) for p in theirs}
    for o in (opt, twin):
        o.add_param_group({"params": torch.nn.Parameter(torch.ones(3)), "muon": False})
        grads(o)
        lists.clear()
        o.step()
        (params, gs, momenta, *rest_args), = lists
        assert [id(p) for p in params] == [id(p) for p in (mine if o is opt else theirs)[:2]] and rest_args[0] == 0.1
        assert all(m is o.state[p]["momentum_buffer"] for p, m in zip(params, momenta)) and float(momenta[0][0, 0]) == 0.5
    for g, h in zip(opt.param_groups, twin.param_groups):
        assert {k: v for k, v in g.items() if k != "params"} == {k: v for k, v in h.items() if k != "params"}
        for p, q in zip(g["params"], h["params"]):
            assert torch.equal(p, q)                         # Adam's moved alike, from the copied state
            assert set(opt.state[p]) == set(twin.state[q]) and all(torch.equal(opt.state[p][k], twin.state[q][k]) for k in opt.state[p])
    assert not torch.equal(opt.param_groups[1]["params"][0], _mixed()[1][0])


def test_convert_group_norm():
    from boostmvsnerfs_amd.config import make_cfg, set_cfg
    from boostmvsnerfs_amd.networks.enerf.cnn import CostRegNet
    from boostmvsnerfs_amd.networks.norm import GroupNorm, convert_group_norm
    for preset, mod, slope in (("enerf_eval", "enerf", False), ("mvsnerf_eval", "mvsnerf", 0.01)):
        set_cfg(make_cfg(preset))
        Network = __import__(f"boostmvsnerfs_amd.networks.{mod}.network", fromlist=["Network"]).Network
        net = Network()
        before = dict(net.named_parameters())
        keys = {k for k in net.state_dict() if "running" not in k and "num_batches" not in k}
        assert convert_group_norm(net, 4) is net
        after = dict(net.named_parameters())
        assert set(after) == set(before) and all(after[k] is before[k] for k in before)
        assert set(net.state_dict()) == keys
        norms = [m for m in net.modules() if isinstance(m, GroupNorm)]
        assert norms and all(m.relu == slope and m.groups == m.weight.numel() // 4 for m in norms)
        assert not any(isinstance(m, nn.modules.batchnorm._BatchNorm) for m in net.modules())
        copy.deepcopy(net)
    with pytest.raises(TypeError, match="whole Network"):
        convert_group_norm(CostRegNet(16))
    with pytest.raises(TypeError, match="whole Network"):
        convert_group_norm(nn.Linear(2, 2))
    set_cfg(make_cfg("enerf_eval"))
    from boostmvsnerfs_amd.networks.enerf.network import Network
    net = Network()
    with pytest.raises(ValueError, match="do not divide"):
        convert_group_norm(net, 3)
    assert not any(isinstance(m, GroupNorm) for m in net.modules())              # refused as a whole


def _regulariser64(m, x, groups):
    """MinCostRegNet with group norms in 64 bits by torch's own operators: (features, depth logits)."""
    def gn(mod, y, relu):
        y = F.group_norm(y, mod.groups, mod.weight.double(), mod.bias.double(), mod.eps)
        return F.relu(y) if relu else y

    def cbr(b, y):
        return gn(b.bn, F.conv3d(y, b.conv.weight.double(), None, b.conv.stride, 1), True)

    def up(u, y):
        return gn(u[1], F.conv_transpose3d(y, u[0].weight.double(), None, stride=2, padding=1, output_padding=1), False)
    s0 = cbr(m.conv0, x)
    s1 = cbr(m.conv2, cbr(m.conv1, s0))
    y = cbr(m.conv4, cbr(m.conv3, s1))
    y = s1 + up(m.conv9, y)
    y = s0 + up(m.conv11, y)
    return F.conv3d(y, m.feat_conv[0].weight.double(), None, 1, 1), F.conv3d(y, m.depth_conv[0].weight.double(), None, 1, 1).squeeze(1)


def _converted(mod="enerf", group_size=8):
    from boostmvsnerfs_amd.networks.norm import convert_group_norm
    Network = __import__(f"boostmvsnerfs_amd.networks.{mod}.network", fromlist=["Network"]).Network
    torch.manual_seed(0)
    return convert_group_norm(Network(), group_size)


def test_another_optimisers_state_is_refused():
    """Groups of one parameter each are as many in Adam's state: not loaded as if they were this one's."""
    from boostmvsnerfs_amd.train import make_optimizer
    net = torch.nn.Sequential(torch.nn.Linear(3, 4), torch.nn.Linear(4, 2))
    adam, muon = make_optimizer(net), make_optimizer(net, optim="muon")
    with pytest.raises(ValueError, match="groups"):
        muon.load_state_dict(adam.state_dict())
    muon.load_state_dict(copy.deepcopy(muon.state_dict()))


@gpu
def test_a_converted_regulariser_against_64_bits():
    """Outputs: 12 layers, each off by fp32 sums of at most 27 x 32 terms (a few 2^-22 of their size): 1e-4 in the 2-norm is
    generous.  Gradients: a z that is off by d flips the ReLU's slope for a share of about d of the values, each flip a whole term:
    sqrt(12 layers x 12 x 2^-22) = 6e-3 of a gradient in the 2-norm; 2e-2 is allowed."""
    from boostmvsnerfs_amd.config import make_cfg, set_cfg
    set_cfg(make_cfg("enerf_eval"))
    m = _converted(group_size=4).cost_reg_0.to(DEV).train()
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, 32, 16, 16, 24, generator=g)
    r = [torch.randn(1, 8, 16, 16, 24, generator=g), torch.randn(1, 16, 16, 24, generator=g)]
    ref = copy.deepcopy(m).cpu()
    want = _regulariser64(ref, x.double(), None)
    sum((a * b.double()).sum() for a, b in zip(want, r)).backward()
    got = m(x.to(DEV))
    for a, b in zip(got, want):
        assert float((a.detach().double().cpu() - b).norm()) <= 1e-4 * float(b.detach().norm())
    sum((a * b.to(DEV)).sum() for a, b in zip(got, r)).backward()
    for (k, p), q in zip(m.named_parameters(), ref.parameters()):
        err = float((p.grad.double().cpu() - q.grad.double()).norm())
        assert err <= 2e-2 * float(q.grad.norm()) + 1e-12, (k, err / float(q.grad.norm()))
    # no mode: evaluation, with and without autograd, is the training forward to fp32 rounding
    with torch.no_grad():
        for a, b in zip(m.eval()(x.to(DEV)), got):
            assert float((a - b.detach()).norm()) <= 1e-5 * float(b.detach().norm())


def _batch(fx, seed):
    b = {k: (v.to(DEV) if torch.is_tensor(v) else v) for k, v in fx.batch().items()}
    g = torch.Generator().manual_seed(seed)
    for i in range(2):
        b[f"rgb_{i}"] = torch.rand(1, b[f"rays_{i}"].shape[1], 3, generator=g).to(DEV)
    return b


@gpu
def test_graphed_and_eager_training_steps_are_the_same(enerf_fx, deterministic):
    """A converted ENeRF with MuonAdam: GraphedTrainStep (eager, captured, replayed steps) against train_step from the same
    state, every gradient, weight and momentum bit for bit; the matrices' update against the formula of ops.muon_step."""
    from boostmvsnerfs_amd import ops
    from boostmvsnerfs_amd.config import set_cfg
    from boostmvsnerfs_amd.train import GraphedTrainStep, NetworkWrapper, make_optimizer, train_step
    set_cfg(tiny_cfg(enerf_fx, "enerf_pretrain"))
    net_a = _converted().to(DEV).train()
    net_b = copy.deepcopy(net_a).train()
    wa, wb = NetworkWrapper(net_a), NetworkWrapper(net_b)
    oa, ob = make_optimizer(net_a, optim="muon"), make_optimizer(net_b, optim="muon")
    step = GraphedTrainStep(wa, oa)
    start = {k: v.clone() for k, v in net_a.state_dict().items()}
    for s in range(6):
        net_b.load_state_dict(copy.deepcopy(net_a.state_dict()))
        ob.load_state_dict(copy.deepcopy(oa.state_dict()))
        before = {k: p.detach().clone() for k, p in net_a.named_parameters()}
        momenta = {k: oa.state[p]["momentum_buffer"].clone() if "momentum_buffer" in oa.state[p] else torch.zeros_like(p)
                   for k, p in net_a.named_parameters()}
        la, _ = step(_batch(enerf_fx, s))
        lb, _ = train_step(wb, ob, _batch(enerf_fx, s))
        assert math.isfinite(float(la)) and float(la) == float(lb)
        named = dict(net_a.named_parameters())
        for (k, p), q in zip(named.items(), net_b.parameters()):
            assert torch.equal(p.grad, q.grad), (s, k)
            assert torch.equal(p, q), (s, k)
        ps = {id(p): k for k, p in named.items()}
        keys = [ps[id(g["params"][0])] for g in oa.param_groups if g["muon"]]
        assert len(keys) == 40
        lists = [before[k] for k in keys], [named[k].grad for k in keys], [momenta[k] for k in keys]
        ops.muon_step(*lists, lr=0.02)
        for k, w, m in zip(keys, lists[0], lists[2]):
            assert torch.equal(w, named[k]) and torch.equal(m, oa.state[named[k]]["momentum_buffer"]), (s, k)
    assert step.stats["eager"] == 3 and step.stats["captures"] == 1 and step.stats["replays"] == 3
    assert sum(float((v - start[k]).abs().max()) > 0 for k, v in net_a.state_dict().items()) > 100


@gpu
@pytest.mark.parametrize("mod,preset", [("enerf", "enerf_eval"), ("mvsnerf", "mvsnerf_eval")])
def test_a_converted_network_renders_and_sees_its_optimiser(mod, preset, enerf_fx):
    """Inference of a converted network (module by module, replayed as a graph from the second call on): repeatable, and a MuonAdam
    step -- which writes the weights behind autograd's back -- reaches every cache of packed weights."""
    from boostmvsnerfs_amd.config import make_cfg, set_cfg
    from boostmvsnerfs_amd.synthetic import clone_batch, make_batch
    from boostmvsnerfs_amd.train import make_optimizer
    cfg = make_cfg(preset)
    if mod == "enerf":
        cfg.enerf.cas_config.volume_planes = [16, 8]
    set_cfg(cfg)
    net = _converted(mod).to(DEV).eval()
    batch = make_batch(64, 96, seed=3) if mod == "enerf" else make_batch(64, 96, render_scales=(1.0,), seed=3, depth_ranges=True)
    key = "rgb_level1" if mod == "enerf" else "rgb_level0"

    def frame():
        with torch.no_grad():
            return net(clone_batch(batch, DEV))[key].clone()
    a = [frame() for _ in range(4)]
    assert torch.isfinite(a[0]).all()
    for b in a[1:]:
        assert float((a[0] - b).abs().max()) <= 1e-5
    opt = make_optimizer(net, optim="muon", muon_lr=0.05)
    for p in net.parameters():
        p.grad = torch.randn_like(p) * 1e-2
    opt.step()
    moved = [frame() for _ in range(3)]
    assert float((moved[0] - a[0]).abs().max()) > 1e-3                            # (0.05 of orthogonal updates)
    twin = _converted(mod).to(DEV).eval()                                           # no caches of the old weights
    twin.load_state_dict(net.state_dict())
    with torch.no_grad():
        fresh = twin(clone_batch(batch, DEV))[key]
    for b in moved:
        assert float((fresh - b).abs().max()) <= 1e-5

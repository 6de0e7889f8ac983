"""GPU: the Muon optimiser over the orthogonalised updates (aadg_amd/muon.py), and the transformer's attention, its gradients and the update
of its matrices run together as `run.py --optimizer muon` runs them."""
import copy
import os

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COEF = (3.4445, -4.7750, 2.0315)


def orthogonal64(u):
    a, b, c = COEF
    x = u.double()
    x = x.t() if u.shape[0] > u.shape[1] else x
    x = x / (x.norm() + 1e-7)
    for _ in range(5):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if u.shape[0] > u.shape[1] else x


def small_net():
    torch.manual_seed(4)
    return nn.Sequential(nn.Conv2d(3, 32, 3, bias=True), nn.Conv2d(32, 32, 3, groups=32), nn.Conv2d(32, 48, 1), nn.Conv2d(48, 2, 1)).cuda()


@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_steps_follow_the_formulas(hip, wd):
    """Three steps against 64-bit restatements.  Matrices: the update has entries of at most ~1 in units of lr 0.2 sqrt(max(shape)); the
    orthogonalisation of these well-conditioned gradients is within 1e-5 of its size, so 1e-4 lr bounds three steps of weights of size
    one in float32 (u = 6e-8).  Others: torch's Adam in float64 on the same gradients."""
    from aadg_amd.muon import Muon, is_matrix
    net = small_net()
    names = [n for n, p in net.named_parameters() if is_matrix(p)]
    assert names == ["0.weight", "2.weight"]                             # not: depthwise filters, the two-row classifier, biases
    lr, mu = 0.01, 0.95
    opt = Muon(net.parameters(), lr=lr, weight_decay=wd)
    ref = {n: p.detach().double().clone() for n, p in net.named_parameters()}
    buf = {n: torch.zeros_like(ref[n]) for n in names}
    others = {n: ref[n].clone().requires_grad_(True) for n in ref if n not in names}
    adam = torch.optim.Adam(list(others.values()), lr=lr, weight_decay=wd)
    for s in range(3):
        torch.manual_seed(s)
        for n, p in net.named_parameters():
            p.grad = torch.randn_like(p) * 1e-3
            if n in others:
                others[n].grad = p.grad.double()
                continue
            g = p.grad.double()
            buf[n] = mu * buf[n] + (1 - mu) * g
            u = ((1 - mu) * g + mu * buf[n]).flatten(1)
            ref[n] = (1 - lr * wd) * ref[n] - lr * 0.2 * max(u.shape) ** 0.5 * orthogonal64(u).view_as(g)
        adam.step()
        opt.step()
    for n, p in net.named_parameters():
        if n in others:
            assert (p.double() - others[n]).abs().max() <= 1e-5 * lr + 4e-7 * ref[n].abs().max(), n
        else:
            assert (p.double() - ref[n]).abs().max() <= 1e-4 * lr * 0.2 * max(p.flatten(1).shape) ** 0.5 + 4e-7 * ref[n].abs().max(), n


def test_state_dict_schedule_and_missing_gradients(hip):
    from aadg_amd.muon import Muon
    net, a = small_net(), None
    twin = copy.deepcopy(net)
    opt = Muon(net.parameters(), lr=0.01)
    sched = torch.optim.lr_scheduler.MultiStepLR(opt, milestones=[1], gamma=0.1)
    x = torch.randn(4, 3, 12, 12, device="cuda")
    for _ in range(2):
        opt.zero_grad(set_to_none=True)
        net(x).square().mean().backward()
        opt.step()
    sched.step()
    assert [g["lr"] for g in opt.param_groups] == pytest.approx([0.001, 0.001])
    twin.load_state_dict(net.state_dict())
    opt2 = Muon(twin.parameters(), lr=0.5)
    opt2.load_state_dict(copy.deepcopy(opt.state_dict()))               # (torch keeps the state's own tensors otherwise: two owners of one momentum)
    for n, o in ((net, opt), (twin, opt2)):
        torch.manual_seed(3)
        for p in n.parameters():
            p.grad = torch.randn_like(p)
        n[2].weight.grad = None                                         # takes no part in this step
        before = n[2].weight.detach().clone()
        o.step()
        assert torch.equal(before, n[2].weight)
    assert all(torch.equal(p, q) for p, q in zip(net.parameters(), twin.parameters()))


def test_refusals(hip):
    from aadg_amd.muon import Muon
    with pytest.raises(hip.AadgError):
        Muon([nn.Parameter(torch.zeros(32, 32))])
    with pytest.raises(hip.AadgError):
        Muon([nn.Parameter(torch.zeros(32, 32, device="cuda", dtype=torch.bfloat16))])
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(eps=0.0), dict(betas=(0.9, 1.0))):
        with pytest.raises(ValueError):
            Muon([nn.Parameter(torch.zeros(32, 32, device="cuda"))], **kw)


@pytest.mark.parametrize("dim,heads,sr", [(64, 1, 4), (64, 2, 2), (40, 5, 1)])
def test_attention_module_matches_float64(hip, dim, heads, sr):
    """The encoder's attention block on the GPU in float32 (own kernels) against the same module in float64 on the CPU (library attention),
    output and the gradients of its input and of every parameter: relative to each tensor's largest value, float32 sums of at most
    B N = 512 terms through four products in a chain, 4 x 512 x 2^-24 = 1.2e-4 at worst."""
    from aadg_amd.models.segformer import Attention
    torch.manual_seed(6)
    m = Attention(dim, heads, sr).cuda()
    ref = copy.deepcopy(m).cpu().double()
    x = torch.randn(2, 256, dim, device="cuda", requires_grad=True)
    xr = x.detach().cpu().double().requires_grad_(True)
    g = torch.randn(2, 256, dim, device="cuda")
    y, yr = m(x, 16, 16), ref(xr, 16, 16)
    y.backward(g)
    yr.backward(g.cpu().double())
    pairs = [(y, yr), (x.grad, xr.grad)] + [(p.grad, q.grad) for p, q in zip(m.parameters(), ref.parameters())]
    floor = max(q.grad.abs().max().item() for q in ref.parameters()) * 1e-3          # the key bias has no gradient but rounding
    for got, want in pairs:
        assert (got.detach().cpu().double() - want).abs().max().item() <= 1.2e-4 * max(want.abs().max().item(), floor)


def test_unsupported_head_width_takes_the_library(hip):
    from aadg_amd.models.segformer import _attend
    q = torch.randn(1, 2, 9, 20, device="cuda")
    assert not hip.attention_supported(q, q, q)
    assert torch.equal(_attend(q, q, q, 0.3), F.scaled_dot_product_attention(q, q, q, scale=0.3))


def test_segformer_training_steps_with_muon(hip):
    """Forward, backward and update of a two-block encoder per stage in bfloat16 autocast: the update of every matrix is the orthogonalised
    gradient (first step: U = (1 - momentum) G + momentum (1 - momentum) G = 0.0975 G; the eps of the norm, 1e-7, is not small beside these), and
    everything stays finite over several steps."""
    from aadg_amd.models.segformer import MIT_B2, SegFormer
    from aadg_amd.muon import Muon, is_matrix
    torch.manual_seed(8)
    net = SegFormer(2, variant=dict(MIT_B2, depths=(1, 2, 1, 1))).cuda()
    opt = Muon(net.parameters(), lr=1e-3)
    x, t = torch.randn(2, 3, 64, 64, device="cuda"), torch.rand(2, 2, 64, 64, device="cuda")
    for step in range(3):
        opt.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            mask, pooled = net(x)
        (F.binary_cross_entropy_with_logits(mask.float(), t) + pooled.square().mean()).backward()
        before = {n: p.detach().clone() for n, p in net.named_parameters()}
        opt.step()
        for n, p in net.named_parameters():
            assert torch.isfinite(p).all()
            if step == 0 and is_matrix(p) and n.startswith("backbone.block2"):
                want = -1e-3 * 0.2 * max(p.flatten(1).shape) ** 0.5 * orthogonal64(0.0975 * p.grad.double().flatten(1))
                got = (p - before[n]).flatten(1).double()
                assert (got - want).abs().max() <= 1e-3 * want.abs().max() + 2e-7 * p.abs().max(), n


def test_search_step_with_muon(hip):
    from aadg_amd import search_dg
    from aadg_amd.config.defaults import get_default_config
    from aadg_amd.muon import Muon
    cfg = get_default_config()
    cfg.defrost()
    cfg.merge_from_file(os.path.join(ROOT, "experiments", "merged_sinkhorn", "segformer_b2_d8.yaml"))
    cfg.TRAIN.BATCH_SIZE = 1
    cfg.DATASET.DG.TRAIN = [1, 2, 3]
    cfg.SEED, cfg.PRINT_FREQ = 1023, 10 ** 9
    cfg.freeze()

    class A(object):
        gpu, workers, distributed = 0, 0, False
        crop_size, backbone_dtype, epoch_items, optimizer = 64, "bf16", 1, "muon"
    st = search_dg.SearchState(0, 1, cfg, A())
    assert isinstance(st.model_optimizer, Muon)
    st.discriminator.synchronize_parameters()
    before = [p.detach().clone() for p in st.model.parameters()]
    *_, losses = st.search_step(0, max_iters=1)
    assert all(torch.isfinite(l).all() for l in losses) and all(torch.isfinite(p).all() for p in st.model.parameters())
    assert sum(not torch.equal(a, b) for a, b in zip(before, st.model.parameters())) > len(before) // 2


def test_groups_given_and_added_are_split_and_checked(hip):
    """A group added later, and groups given as dicts, are split and checked like the parameters of the constructor."""
    from aadg_amd.muon import Muon, is_matrix
    net, late = small_net(), nn.Sequential(nn.Conv2d(2, 32, 3, bias=True), nn.Conv2d(32, 32, 3, groups=32), nn.Linear(32, 40)).cuda()
    a, b = copy.deepcopy(net), copy.deepcopy(late)
    one = Muon([p for m in (a, b) for p in m.parameters()], lr=0.01)
    two = Muon(net.parameters(), lr=0.01)
    two.add_param_group(dict(params=late.parameters(), lr=0.02))
    three = Muon([dict(params=list(copy.deepcopy(net).parameters()), weight_decay=0.1), dict(params=copy.deepcopy(late)[2].weight, lr=0.02)], lr=0.01)
    for opt in (one, two, three):
        for g in opt.param_groups:
            assert all(is_matrix(p) == g["matrices"] for p in g["params"])
    assert [(g["lr"], g["matrices"], len(g["params"])) for g in two.param_groups] == [(0.01, True, 2), (0.01, False, 6), (0.02, True, 2), (0.02, False, 4)]
    assert [(g["lr"], g["weight_decay"], g["matrices"]) for g in three.param_groups] == [(0.01, 0.1, True), (0.01, 0.1, False), (0.02, 0.0, True)]
    for g in two.param_groups[2:]:
        g["lr"] = 0.01
    for m, n in ((a, net), (b, late)):
        for p, q in zip(m.parameters(), n.parameters()):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
    one.step()
    two.step()
    for m, n in ((a, net), (b, late)):
        assert all(torch.equal(p, q) for p, q in zip(m.parameters(), n.parameters()))
    # the group's own word: everything to Adam
    table = nn.Parameter(torch.zeros(64, 32, device="cuda"))
    two.add_param_group(dict(params=[table], matrices=False))
    assert two.param_groups[-1]["matrices"] is False
    bias = lambda **kw: nn.Parameter(torch.zeros(32, **kw))                                      # noqa: E731
    with pytest.raises(ValueError):
        two.add_param_group(dict(params=[bias(device="cuda")], matrices=True))
    with pytest.raises(ValueError):
        two.add_param_group(dict(params=[bias(device="cuda")], lr=-1.0))
    with pytest.raises(ValueError):
        two.add_param_group(dict(params=[bias(device="cuda")], steps=0))
    with pytest.raises(ValueError):
        two.add_param_group(dict(params=[table]))                                           # twice
    for p in (bias(), bias(device="cuda", dtype=torch.bfloat16)):
        with pytest.raises(hip.AadgError):
            two.add_param_group(dict(params=[p]))
    with pytest.raises(ValueError):
        Muon([table.detach()])                                                              # nothing to train
    assert len(two.param_groups) == 5


def test_matrices_past_one_call_of_the_library(hip):
    """More matrices than one call takes; a matrix longer than the library takes has Adam's update."""
    from aadg_amd.muon import Muon, is_matrix
    torch.manual_seed(12)
    many = [nn.Parameter(torch.randn(16, 17, device="cuda")) for _ in range(4100)]
    table = nn.Parameter(torch.randn((1 << 16) + 1, 16, device="cuda"))
    assert is_matrix(many[0]) and not is_matrix(table)
    opt = Muon(many + [table], lr=0.01)
    before = [p.detach().clone() for p in many]
    for p in many + [table]:
        p.grad = torch.randn_like(p)
    start = table.detach().clone()
    opt.step()
    for i in (0, 4095, 4096, 4099):                                         # U = 0.0975 G
        want = -0.01 * 0.2 * 17 ** 0.5 * orthogonal64(0.0975 * many[i].grad.double())
        assert ((many[i] - before[i]).double() - want).abs().max() <= 1e-4 * want.abs().max() + 2.0 ** -23 * before[i].abs().max()
    # Adam's first step: lr g / (|g| + eps) up to rounding
    assert ((table - start) + 0.01 * table.grad.sign()).abs().max() <= 2.0 ** -23 * start.abs().max() + 0.01 * 1e-8 / table.grad.abs().min()
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[nn.Parameter(torch.zeros((1 << 16) + 1, 16, device="cuda"))], matrices=True))


def test_a_captured_step_is_refused(hip, monkeypatch):
    """the learning rate and Adam's step count are host values: a captured step would repeat them on every replay"""
    from aadg_amd.muon import Muon
    net = small_net()
    opt = Muon(net.parameters(), lr=0.01)
    for p in net.parameters():
        p.grad = torch.randn_like(p)
    before = [p.detach().clone() for p in net.parameters()]
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(hip.AadgError):
            opt.step()
    assert all(torch.equal(a, b) for a, b in zip(before, net.parameters())) and not opt.state
    opt.step()
    assert not any(torch.equal(a, b) for a, b in zip(before, net.parameters()))


def test_named_parameters(hip):
    from aadg_amd.muon import Muon, is_matrix
    net = small_net()
    twin = copy.deepcopy(net)
    opt, plain = Muon(net.named_parameters(), lr=0.01), Muon(twin.parameters(), lr=0.01)
    assert sum((g["param_names"] for g in opt.param_groups), []) == sorted(dict(net.named_parameters()), key=lambda n: not is_matrix(net.get_parameter(n)))
    for p, q in zip(net.parameters(), twin.parameters()):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    opt.step()
    plain.step()
    assert all(torch.equal(p, q) for p, q in zip(net.parameters(), twin.parameters()))


def test_a_refused_group_leaves_the_optimizer_as_it_was(hip):
    from aadg_amd.muon import Muon
    w = lambda: nn.Parameter(torch.zeros(32, 32, device="cuda"))                                 # noqa: E731
    opt = Muon([w()])
    for params, error in (([w(), torch.zeros(32, device="cuda", requires_grad=True) * 2], ValueError), ({w(), w()}, TypeError), ([w(), "bias"], TypeError)):
        with pytest.raises(error):
            opt.add_param_group(dict(params=params))
        assert len(opt.param_groups) == 1

"""CPU: the choice of the optimiser (`run.py --optimizer`) and which parameters get orthogonalised updates."""
import pytest
import torch
import torch.nn as nn


def test_run_py_offers_the_optimizers():
    import run
    assert run.parse_args(["--cfg", "x.yaml"]).optimizer == "adam"
    assert run.parse_args(["--cfg", "x.yaml", "--optimizer", "muon"]).optimizer == "muon"
    with pytest.raises(SystemExit):
        run.parse_args(["--cfg", "x.yaml", "--optimizer", "sgd"])


def test_scheduler_default_is_adam_and_unknown_is_refused():
    from aadg_amd.config.defaults import get_default_config
    from aadg_amd.scheduler import get_optimizer_scheduler
    cfg, net = get_default_config(), nn.Linear(20, 20)
    assert type(get_optimizer_scheduler(net, net, cfg)[0]) is torch.optim.Adam
    with pytest.raises(ValueError):
        get_optimizer_scheduler(net, net, cfg, "sgd")


def test_which_parameters_are_matrices():
    from aadg_amd.muon import is_matrix
    yes = [(64, 64), (16, 16), (64, 3, 7, 7), (64, 16, 1, 1)]
    no = [(64,), (), (2, 768), (64, 1, 3, 3), (15, 400), (64, 8), (2, 256, 1, 1)]
    assert all(is_matrix(torch.zeros(s)) for s in yes) and not any(is_matrix(torch.zeros(s)) for s in no)


def test_sizes_outside_the_library_stay_with_adam():
    from aadg_amd.muon import is_matrix
    no = [(0, 64), (64, 0), ((1 << 16) + 1, 16), (16, (1 << 16) + 1), (1 << 15, (1 << 13) + 1)]
    assert not any(is_matrix(torch.empty(s, device="meta")) for s in no)
    assert all(is_matrix(torch.empty(s, device="meta")) for s in [(1 << 16, 16), (16, 1 << 16), (1 << 15, 1 << 13)])

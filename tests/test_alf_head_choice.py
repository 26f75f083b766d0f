"""not-gpu: which loss each phase of run_alf.py fits the last level with, and the choices that contradict each other."""
import os
import sys

import numpy as np
import pytest
import torch

from neuron_interpolation_model_fusion_amd.fusion_algorithms import ALFusion
from tests.test_alf_head_loss import _config, _models

SCRIPTS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'main_scripts', 'run_individual_algorithms')


@pytest.fixture
def run_alf(monkeypatch, tmp_path):
    """run(*flags) -> [(head_loss, use_kd_on_head, kd_temperature, skipped levels)] of its fits, which are not made."""
    monkeypatch.syspath_prepend(SCRIPTS)
    import _common as c
    import run_alf as script
    models = _models()
    fits = []
    monkeypatch.setattr(c, 'load_models', lambda *a: models)
    monkeypatch.setattr(c, 'fusion_dataset', lambda *a: None)
    monkeypatch.setattr(c, 'fusion_samples', lambda *a, **k: (torch.zeros(4, 64), torch.zeros(4, dtype=torch.long)))
    monkeypatch.setattr(c, 'num_classes_of', lambda *a: 10)
    monkeypatch.setattr(c, 'report', lambda *a: None)
    monkeypatch.setattr(script, 'get_classifier_head_weights', lambda *a, **k: np.ones((2, 10)))
    monkeypatch.setattr(torch, 'save', lambda *a, **k: None)

    def fuse(self, cfg):
        self._config_check(cfg)
        fits.append((cfg.head_loss, cfg.use_kd_on_head, cfg.kd_temperature, cfg.skip_levels))
    monkeypatch.setattr(ALFusion, 'fuse', fuse)

    def run(*flags):
        monkeypatch.setattr(sys, 'argv', ['run_alf.py', '--model_savedir', str(tmp_path), '--num_fusion_samples', '4', '--num_models', '2',
                                          '--device', 'cpu', *flags])
        fits.clear()
        script.main()
        return list(fits)
    return run


@pytest.mark.parametrize('kl', [False, True])
@pytest.mark.parametrize('loss', ['match', 'cross_entropy'])
def test_the_distillation_phase_distils(run_alf, loss, kl):
    flags = ['--use_kl_kd_on_head'] if kl else []
    fits = run_alf('--head_loss', loss, '--run_last_layer_kd', '--kd_temperature', '3', *flags)
    assert [f[:2] for f in fits[:3]] == [(loss, False)] * 3 and len(fits) == 4
    assert fits[3] == ('match', kl, 3.0, [0])


def test_the_distillation_phase_keeps_top_logits(run_alf):
    fits = run_alf('--head_loss', 'top_logits', '--run_last_layer_kd', '--kd_temperature', '3')
    assert [f[:3] for f in fits] == [('top_logits', False, 3.0)] * 4 and fits[3][3] == [0]


def test_two_distillations_at_once_are_refused(run_alf, capsys):
    with pytest.raises(SystemExit):
        run_alf('--head_loss', 'top_logits', '--run_last_layer_kd', '--use_kl_kd_on_head')
    assert '--use_kl_kd_on_head' in capsys.readouterr().err


@pytest.mark.parametrize('loss', ['cross_entropy', 'top_logits'])
def test_a_loss_on_the_head_and_kd_on_head_contradict(loss):
    with pytest.raises(ValueError, match='use_kd_on_head'):
        ALFusion(_models()).fuse(_config(torch.zeros(4, 64), head_loss=loss, kd_temperature=2.0, use_kd_on_head=True))


def _hook(*args):
    return None


@pytest.mark.parametrize('watch', [
    lambda net, head: head.register_forward_hook(_hook), lambda net, head: head.register_forward_pre_hook(_hook),
    lambda net, head: head.register_full_backward_hook(_hook), lambda net, head: head.register_full_backward_pre_hook(_hook),
    lambda net, head: net.register_forward_hook(_hook), lambda net, head: net.register_forward_pre_hook(_hook),
    lambda net, head: net.register_full_backward_hook(_hook)])
@pytest.mark.parametrize('loss', ['cross_entropy', 'top_logits'])
def test_hooks_that_the_loss_would_pass_by_are_refused(loss, watch):
    """The loss takes the head's input and weight: the head and the level's Sequential are not called."""
    models = _models()
    network = models[0].get_ordered_trainable_named_levels[-1].network
    handle = watch(network, network[-1])
    cfg = _config(torch.zeros(4, 64), head_loss=loss, kd_temperature=2.0)
    with pytest.raises(ValueError, match='hooks'):
        ALFusion(models).fuse(cfg)
    with pytest.raises(ValueError, match='hooks'):  # on the model that is fused into
        ALFusion(_models()).fuse(cfg, models[0])
    handle.remove()
    ALFusion(models)._config_check(cfg)


def test_a_head_with_a_forward_of_its_own_is_refused():
    class Scaled(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    class Twice(torch.nn.Sequential):
        def forward(self, x):
            return 2 * super().forward(x)
    for network in (Scaled(4, 3), torch.nn.Sequential(torch.nn.Flatten(), Scaled(4, 3)), Twice(torch.nn.Flatten(), torch.nn.Linear(4, 3))):
        with pytest.raises(ValueError, match='forward of its own'):
            ALFusion._body_and_head(network)
    wrapped = torch.nn.Linear(4, 3)
    wrapped.forward = lambda x: 2 * torch.nn.Linear.forward(wrapped, x)
    with pytest.raises(ValueError, match='forward of its own'):
        ALFusion._body_and_head(wrapped)
    body, head = ALFusion._body_and_head(torch.nn.Sequential(torch.nn.Flatten(), torch.nn.Linear(4, 3)))
    assert len(body) == 1 and head.out_features == 3


@pytest.mark.parametrize('y', [torch.tensor([0.0, 1.5, 2.0, 3.0]), torch.tensor([0.0, float('nan'), 1.0, 2.0]),
                               torch.tensor([0.0, float('inf'), 1.0, 2.0])])
def test_labels_that_are_no_whole_numbers_are_refused(y):
    """They travel as float rows and are cut to whole numbers on the way into the loss."""
    with pytest.raises(ValueError, match='labels must'):
        ALFusion(_models()).fuse(_config(torch.zeros(4, 64), head_loss='cross_entropy', y=y))
    ALFusion(_models())._config_check(_config(torch.zeros(4, 64), head_loss='cross_entropy', y=torch.tensor([0.0, 9.0, 1.0, 2.0])))

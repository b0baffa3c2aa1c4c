"""Refusals that the host sides of the C entry points make before anything reaches a device, and host arithmetic of the
operators for expert layers and 8-bit formats."""
import pytest
import torch

from vitpose_amd import _lib, optim

ERR_ARG = -1


def adamw8(**over):
    a = dict(p=64, g=64, m=64, ms=64, r=64, rs=64, half=None, start=64, length=64, scale=64, wd=64, state=64, nchunks=1, numel=128,
             state_numel=128, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, step=1, partials=None, npartials=0, max_norm=0.0,
             grad_scale=1.0, noise=0)
    a.update(over)
    return _lib.lib().vp_adamw8_step(*a.values(), None)


@pytest.mark.parametrize('over', [dict(p=None), dict(g=None), dict(m=None), dict(rs=None), dict(start=None), dict(state=None),
                                  dict(step=0), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(nchunks=-1), dict(numel=-1),
                                  dict(state_numel=100), dict(p=72), dict(g=68), dict(m=65), dict(half=66), dict(npartials=257),
                                  dict(npartials=3), dict(npartials=3, partials=64, max_norm=0.0)])
def test_adamw8_refuses_on_the_host(over):
    assert adamw8(**over) == ERR_ARG


def test_adamw8_with_an_empty_table_does_nothing():
    assert adamw8(nchunks=0, p=None, g=None) == 0


@pytest.mark.parametrize('over', [dict(partials=None), dict(n=0), dict(n=257), dict(x=None), dict(x=72), dict(nchunks=-1)])
def test_sumsq_chunks_f64_refuses_on_the_host(over):
    a = dict(x=64, start=64, length=64, nchunks=1, numel=4, partials=64, n=1)
    a.update(over)
    assert _lib.lib().vp_sumsq_chunks_f64(*a.values(), None) == ERR_ARG


def test_adamw8_needs_a_device():
    st = optim.new_state8(128, 'cpu')
    with pytest.raises(RuntimeError):
        optim.adamw8_step(torch.zeros(4), torch.zeros(4), st, (), lr=1e-3, step=1, noise=0)
    with pytest.raises(ValueError):
        optim.new_state8(100, 'cpu')


def test_noise_keys_differ_by_step_and_seed():
    keys = {optim.noise_key(s, t) for s in range(8) for t in range(1, 129)}
    assert len(keys) == 8 * 128 and all(0 <= k < 1 << 31 for k in keys)

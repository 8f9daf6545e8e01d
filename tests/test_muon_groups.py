"""Muon's groups: one that is refused leaves the optimizer as it was (no GPU needed)."""
import importlib

import pytest
import torch


def test_a_vector_is_refused_before_it_is_added():
    O = importlib.import_module('dcss-auto_amd.optim')
    matrix, more, vector = (torch.nn.Parameter(torch.zeros(s)) for s in ((4, 5), (2, 3), (5,)))
    opt = O.Muon([matrix])
    for group in (dict(params=[vector]), dict(params=vector), dict(params=[more, vector]), dict(params=iter([more, vector])),
                  dict(params=[torch.nn.Parameter(torch.tensor(1.0))])):
        with pytest.raises(ValueError, match='two dimensions'):
            opt.add_param_group(group)
        assert len(opt.param_groups) == 1 and opt.param_groups[0]['params'] == [matrix]
    with pytest.raises(ValueError, match='momentum'):
        opt.add_param_group(dict(params=[more], momentum=0.5))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=iter([more]), lr=0.5))
    assert opt.param_groups[1]['lr'] == 0.5 and opt.param_groups[1]['params'] == [more]
    named = O.Muon([('a', matrix)])
    with pytest.raises(ValueError, match='two dimensions'):
        named.add_param_group(dict(params=[('v', vector)]))
    assert len(named.param_groups) == 1
    named.add_param_group(dict(params=[('b', more)]))
    assert named.param_groups[1]['params'] == [more]

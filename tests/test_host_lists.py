"""npn_native.check_lists without a GPU."""
import types

import pytest
import torch

import npn_native

HERE = types.SimpleNamespace(index=-1)  # what a CPU tensor's get_device says


def test_every_layer_has_the_first_one_s_shape():
    """K's pages and V's have the same number of bytes: a list's later entries are checked by shape as its first is."""
    k, v = torch.empty(3, 2, 16, 256, dtype=torch.int8), torch.empty(3, 2, 256, 16, dtype=torch.int8)
    rows = torch.empty(3, 2)
    spec = lambda ts, shape=k.shape: (ts, "cache_ks", torch.int8, tuple(shape))  # noqa: E731
    out = npn_native.check_lists(HERE, spec([k, k.clone(), k.clone()]), (4 * [rows], "k_scales", torch.float32, (3, 2)))
    assert [len(a.pointers) for a in out] == [3, 4]
    for bad in ([k, v], [k, k, k.reshape(3, 2, 32, 128)], [k, k.reshape(-1)], [v, k], [k, k[:2]], [k, k.float()],
                [k, v.transpose(2, 3)]):
        with pytest.raises((RuntimeError, TypeError)):
            npn_native.check_lists(HERE, spec(bad))
    with pytest.raises(RuntimeError):
        npn_native.check_lists(HERE, ([rows, rows.reshape(2, 3)], "k_scales", torch.float32, (3, 2)))


def test_layers_of_a_number_of_elements_have_any_shape():
    x = torch.empty(4, 6)
    npn_native.check_lists(HERE, ([x, x.reshape(-1), x.reshape(2, 12)], "records", torch.float32, 24))
    with pytest.raises((RuntimeError, TypeError)):
        npn_native.check_lists(HERE, ([x, torch.empty(23)], "records", torch.float32, 24))

"""The 64-bit restatement of the operators on rows of logits (tests/logits_ref.py) on cases worked out by
hand, and the C entry points' refusals that need no device."""
import ctypes as C

import numpy as np
import pytest

import logits_ref as ref


def test_order_of_ties_and_short_rows():
    z = np.array([1.0, 3.0, -np.inf, 3.0, np.nan, 0.0, -0.0])
    v, i, lse = ref.top(z, 6, 1.0)
    assert i.tolist() == [1, 3, 0, 5, 6, -1]
    assert v.tolist() == [3.0, 3.0, 1.0, 0.0, 0.0, -np.inf]
    assert abs(lse - np.log(2 * np.exp(3) + np.exp(1) + 2)) < 1e-12


def test_mask_words_round_trip():
    bits = np.random.default_rng(0).random(131) < 0.5
    assert np.array_equal(ref.unpack_mask(ref.pack_mask(bits), 131), bits)


def test_distillation_against_its_definition():
    z, ids, t = np.log([1.0, 2.0, 5.0, 2.0]), [2, 1], np.log([3.0, 1.0])
    loss, (L, off), g, _ = ref.distill(z, ids, t, None, 1.0)
    q, p = np.array([0.1, 0.2, 0.5, 0.2]), np.array([0.75, 0.25])
    assert abs(loss - (p * np.log(p / q[[2, 1]])).sum()) < 1e-12 and off == 1.0 and abs(L - np.log(10)) < 1e-12
    assert np.allclose(g, [0.1, 0.2 - 0.25, 0.5 - 0.75, 0.2])
    loss, (L, off), g, _ = ref.distill(z, ids, t, np.log(8.0), 1.0)  # p = 3/8, 1/8 and 1/2 for the rest
    want = 0.375 * np.log(0.375 / 0.5) + 0.125 * np.log(0.125 / 0.2) + 0.5 * np.log(0.5 / 0.3)
    assert abs(loss - want) < 1e-12
    assert np.allclose(g, [0.1 * (1 - 0.5 / 0.3), 0.2 - 0.125, 0.5 - 0.375, 0.2 * (1 - 0.5 / 0.3)])
    assert abs(g.sum()) < 1e-12


def test_cuts_of_sampling():
    z = np.log([0.5, 0.25, 0.125, 0.125])
    unit = ref.GRID
    assert ref.sample_weights(z, 1.0, 0, 1.0, 0.0).tolist() == [unit, unit / 2, unit / 4, unit / 4]
    assert ref.sample_weights(z, 1.0, 3, 1.0, 0.0).tolist() == [unit, unit / 2, unit / 4, 0]
    assert ref.sample_weights(z, 1.0, 0, 0.6, 0.0).tolist() == [unit, unit / 2, 0, 0]
    assert ref.sample_weights(z, 1.0, 0, 1.0, 0.3).tolist() == [unit, unit / 2, 0, 0]
    assert ref.sample_weights(z, 0.0, 0, 1.0, 0.0).tolist() == [unit, 0, 0, 0]
    assert ref.sample_weights(z, 1.0, 0, 0.0, 0.0).tolist() == [unit, 0, 0, 0]
    assert ref.sample_weights(z[:0], 1.0, 0, 1.0, 0.0).tolist() == []


def test_entry_points_refuse_a_missing_context():
    from winrapids_b200 import _lib, build

    build.build()
    L = _lib.lib()
    x, t, p = _lib.Logits(), _lib.Teacher(), _lib.Sampling()
    assert L.tbgb_top_logits(None, C.byref(x), 1, 1.0, None, 0, None, None, None, None) == 7
    assert L.tbgb_distill_loss(None, C.byref(x), C.byref(t), None, None, None) == 7
    assert L.tbgb_distill_grad(None, C.byref(x), C.byref(t), None, None, None, 0, None) == 7
    assert L.tbgb_distill_step(None, C.byref(x), C.byref(t), None, None, None, None, 0, None) == 7
    assert L.tbgb_sample_tokens(None, C.byref(x), None, C.byref(p), None, 0, None, None, None) == 7


@pytest.mark.parametrize("name,size", [("Logits", 40), ("Teacher", 56), ("Sampling", 48)])
def test_struct_sizes_follow_the_header(name, size):
    from winrapids_b200 import _lib

    assert C.sizeof(getattr(_lib, name)) == size

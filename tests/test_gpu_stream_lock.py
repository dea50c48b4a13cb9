"""A streamed dense shard whose rows cannot be page-locked in place: the driver
refuses it for memory that exists (the rows stay pageable, the results the
same), or the locking fails (the load does)."""
from __future__ import annotations

import pytest

import distlr_amd as dlr
from test_gpu_parity import assert_same_weights

pytestmark = pytest.mark.gpu

D, ROWS, B = 256, 1000, 300  # four batches, the last wraps to row 0


def epochs(eng, dd, residency, fault=dlr.FAULT_NONE, n=3):
    eng.set_residency(residency)
    eng.set_fault(fault)
    nb = eng.load_train_dense(dd, B)
    eng.set_weights(dlr.init_weight(D))
    for _ in range(n):
        for b in range(nb):
            eng.train_step(b, 0.05)
    return eng.get_weights()


def test_pageable_rows_stream_to_the_same_bits():
    one, two = (dlr.DenseDataset.generate(ROWS, D, seed=s, stream=1) for s in (21, 22))
    eng = dlr.Engine(D)
    try:
        with pytest.raises(dlr.DLRError):
            eng.train_host_locked()  # no shard
        want = [epochs(eng, dd, dlr.RESIDENCY_DEVICE) for dd in (one, two)]
        assert eng.train_host_locked() is False
        for fault in (dlr.FAULT_LOCK_REFUSED, dlr.FAULT_NONE):  # as the driver decides
            for dd, w in ((one, want[0]), (two, want[1]), (one, want[0])):  # reloads
                assert_same_weights(epochs(eng, dd, dlr.RESIDENCY_STREAM, fault), w)
                assert eng.train_residency() == dlr.RESIDENCY_STREAM
                assert not (fault and eng.train_host_locked())
        assert_same_weights(epochs(eng, two, dlr.RESIDENCY_DEVICE), want[1])
    finally:
        eng.close()


def test_a_sparse_copy_is_page_locked():
    ds = dlr.Dataset.generate(500, 4096, 10, seed=3, stream=1)
    eng = dlr.Engine(4096)
    try:
        eng.set_residency(dlr.RESIDENCY_STREAM)
        eng.load_train(ds, 100)
        assert eng.train_residency() == dlr.RESIDENCY_STREAM and eng.train_host_locked()
    finally:
        eng.close()


def test_a_locking_that_fails_fails_the_load():
    dd = dlr.DenseDataset.generate(ROWS, D, seed=23, stream=1)
    eng = dlr.Engine(D)
    try:
        want = epochs(eng, dd, dlr.RESIDENCY_DEVICE)
        with pytest.raises(dlr.DLRError) as e:
            epochs(eng, dd, dlr.RESIDENCY_STREAM, dlr.FAULT_LOCK_FAILED)
        assert e.value.code == -4 and "hipHostRegister" in str(e.value)  # DLR_E_HIP
        with pytest.raises(dlr.DLRError):
            eng.train_residency()  # nothing is loaded
        assert_same_weights(epochs(eng, dd, dlr.RESIDENCY_STREAM), want)  # the fault lasts one load
    finally:
        eng.close()

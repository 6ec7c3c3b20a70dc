"""Requests with extended fields on the host: found wherever they stand, and never dropped."""
from collections import deque
from types import SimpleNamespace

import numpy as np
import pytest

from conftest import pkg

NS = pkg()
packing = pkg("packing")
history = pkg("history")
SP, EP = NS.SamplingParams, NS.ExtendedSamplingParams
FIELDS = (("presence_penalty", 1.0), ("frequency_penalty", -0.5), ("logit_bias", {5: -100.0}))


def _plain(kind):
    fields = dict(temperature=1.0, top_p=1.0, top_k=-1, repetition_penalty=1.0)
    return SP() if kind == "dataclass" else SimpleNamespace(**fields)


@pytest.mark.parametrize("field,value", FIELDS)
@pytest.mark.parametrize("kind", ["namespace", "dataclass"])
@pytest.mark.parametrize("at", [0, 1, 4])
def test_every_request_is_looked_at(kind, field, value, at):
    """A field that only one object of a type has counts wherever that object stands in the batch."""
    params = [_plain(kind) for _ in range(5)]
    assert not packing.wants_processing(params)
    setattr(params[at], field, value)
    assert packing.wants_processing(params)
    assert packing.wants_processing(tuple(params)) and packing.wants_processing(deque(params))
    setattr(params[at], field, None)
    assert not packing.wants_processing(params)


class _Slots:
    __slots__ = ("temperature", "top_p", "top_k", "repetition_penalty", "logit_bias")


def test_types_of_every_make_are_looked_at():
    class Computed(SP):
        @property
        def presence_penalty(self):
            return 0.25

    class Found(SP):
        def __getattr__(self, name):
            if name == "frequency_penalty":
                return 0.25
            raise AttributeError(name)

    bare, biased = _Slots(), _Slots()
    biased.logit_bias = {1: 2.0}
    assert not packing.wants_processing([bare, SP()])
    for params in ([bare, biased], [biased, bare], [SP(), Computed()], [SP(), Found()]):
        assert packing.wants_processing(params)


@pytest.mark.parametrize("seeds", [[None] * 4, [None, 3, None, 2**64 - 1], [0] * 4])
def test_row_records_are_those_of_one_request_at_a_time(seeds):
    params = [SP(temperature=t, top_k=k, seed=s) for t, k, s in zip((0.0, 0.5, 1.0, -1.0), (-1, 0, 49, 50), seeds)]
    got = packing.derive_rows(params, 50, [0, 1, 2, 3])
    want = np.array([packing.derive_row(p, 50, n) for n, p in enumerate(params)], dtype=packing.ROW_DTYPE)
    assert got.tobytes() == want.tobytes()

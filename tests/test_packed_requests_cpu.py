"""Packing for Sampler.sample_packed refuses requests with fields that it would drop."""
import numpy as np
import pytest

from conftest import pkg

NS = pkg()
packing = pkg("packing")
history = pkg("history")
SP, EP = NS.SamplingParams, NS.ExtendedSamplingParams


def _biased():
    p = SP()
    p.logit_bias = {3: -np.inf}
    return p


EXTENDED = [EP(presence_penalty=0.5), EP(frequency_penalty=-0.5), EP(logit_bias={3: 1.0}), _biased()]


@pytest.mark.parametrize("which", range(len(EXTENDED)))
@pytest.mark.parametrize("at", [0, 2])
def test_pack_refuses_what_it_would_drop(which, at):
    params = [SP(), EP(repetition_penalty=1.2), SP()]
    packed = packing.pack(params, [[1], [2, 3], []], 10, sms=4)
    assert packed.offsets.tolist() == [0, 0, 2, 2] and packed.ids.tolist() == [2, 3]
    params[at] = EXTENDED[which]
    with pytest.raises(ValueError, match="process_logits"):
        packing.pack(params, [[1], [2, 3], []], 10, sms=4)


@pytest.mark.parametrize("store", ["HistoryStore", "PagedHistoryStore"])
@pytest.mark.parametrize("which", range(len(EXTENDED)))
def test_the_stores_refuse_it_too(store, which):
    st = object.__new__(getattr(NS, store))  # its pools need a GPU, the check does not
    with pytest.raises(ValueError, match="process_logits"):
        st.pack([SP(), EXTENDED[which]], [0, 1])


def test_fields_that_ask_for_nothing_are_no_reason():
    for p in (EP(), EP(presence_penalty=0.0, frequency_penalty=0.0, logit_bias={}), EP(logit_bias=None)):
        assert packing.pack([p], [[]], 10).num_rows == 1

"""Slots without a row of logits, or that are none: Model.sample_rows and Model.sample_tokens say which call and which slot."""
import pytest

from ai00_server_b200 import capi, runtime, synth

pytestmark = pytest.mark.gpu


def test_slots_without_rows():
    m = runtime.Model(synth.make_st("tiny6", 0), max_batch=3, token_chunk_size=16)
    m.state.load(m.state.init(), 0)
    m.infer_raw([0], [1], [5], [capi.OPTION_LAST])
    for name, call in (("sample_rows", lambda slots: m.sample_rows(slots)), ("sample_tokens", lambda slots: m.sample_tokens(slots, [0.5] * len(slots)))):
        call([0, 0])
        for slots, text in (([0, 2], f"{name}: slot 2 has produced no logits row yet"), ([0, 3], f"{name}: slot out of range"), ([-1], f"{name}: slot out of range")):
            with pytest.raises(capi.B200Error) as ei:
                call(slots)
            assert ei.value.code == capi.ERR_STATE and text in str(ei.value)
    m.close()

"""A decode session that is kept while its slots' sequences change: each step takes the adapters that they have by then."""
import numpy as np
import pytest

import tiny
from test_gpu_requests import adapted_engine, logits_of, setting  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("before,after", [(None, "one"), ("one", None), ("one", "two")])
def test_a_slot_that_was_opened_again_with_another_adapter(setting, before, after):  # noqa: F811
    from foundry_b200 import SequenceStep
    V = setting["cfg"]["vocab_size"]
    engine = adapted_engine(setting, max_slots=1)
    session = None
    for name in (before, after, before):
        prompt = tiny.random_tokens(5, 12, V)
        slot = engine.open_sequence(name) if name else engine.open_sequence()
        first = int(np.argmax(engine.step([SequenceStep(slot, prompt, [11])])[0].cpu().numpy()))
        session = session or engine.decode_session([slot])
        assert session.slots == [slot]
        tokens, said = [first], []
        for _ in range(5):
            said += tokens
            tokens = session.step_host(tokens)
            got = session.logits()[0].cpu().numpy()
            tiny.assert_logits_close(got[None], logits_of(setting, name, prompt + said)[-1:], "float32")
        engine.close_sequence(slot)

"""The checks and the first call of sample_rows (yalm_b200/sampling.py), which need no GPU."""
import threading

import pytest

from yalm_b200 import YalmB200Error, sampling


def test_a_first_call_while_another_sets_up(monkeypatch):
    """A call from a second thread at every step of the first one's setting up finds all that it needs or sets up itself."""
    import torch
    x, coin, tokens = torch.zeros(1, 8), torch.zeros(1), torch.zeros(1, dtype=torch.int32)
    seen = []

    def call():
        try:
            sampling.sample_rows(x, coin, tokens)
        except Exception as e:
            seen.append(e)

    class Codes(dict):
        def __setitem__(self, k, v):
            if threading.current_thread() is threading.main_thread():
                t = threading.Thread(target=call)
                t.start()
                t.join()
            super().__setitem__(k, v)

    monkeypatch.setattr(sampling, "_codes", Codes())
    monkeypatch.setattr(sampling, "_stream", None)
    call()
    # without a GPU the library refuses what is not memory of one, and so it does with one
    assert len(seen) >= 3 and all(isinstance(e, YalmB200Error) for e in seen), seen


@pytest.mark.parametrize("bad", [dict(coin=None), dict(tokens=None)])
def test_what_has_to_be_given(bad):
    import torch
    a = dict(coin=torch.zeros(1), tokens=torch.zeros(1, dtype=torch.int32))
    a.update(bad)
    with pytest.raises(ValueError):
        sampling.sample_rows(torch.zeros(1, 8), **a)

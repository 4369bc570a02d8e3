"""Where the stochastic 8-bit float layer runs, without a GPU: a recorder stands in for the library, so nothing is launched."""
import pytest
import torch

import quantised_bayesian_nets_amd as q
from quantised_bayesian_nets_amd import _lib, fp8, models_f32


class Recorder:
    """Answers every entry with success and notes its name."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append(name)
            return 0
        return entry


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: r)
    monkeypatch.setattr(_lib, "current_stream", lambda: None)
    return r


@pytest.mark.parametrize("kind", [fp8.Linear, models_f32.Linear])
def test_a_cpu_input_reaches_no_kernel(recorder, kind):
    m = kind(6, 4, True)
    with q.mc_context(3, 1):
        for call in (lambda: m(torch.zeros(1, 2, 6)), lambda: m(torch.zeros(1, 2, 6), eps=torch.zeros(3, 24)), lambda: m.sampled(torch.device("cpu"))):
            with pytest.raises(RuntimeError, match="MI355X only"):
                call()
    assert recorder.calls == [] and m._sigma is None


def test_a_cpu_operand_in_blocks_reaches_no_kernel(recorder):
    x = q.F8Tensor(torch.zeros(1, 2, 128, dtype=torch.float8_e4m3fn), torch.full((1, 2, 4), 127, dtype=torch.uint8), 6, 1)
    with q.mc_context(3, 1), pytest.raises(RuntimeError, match="MI355X only"):
        fp8.Linear(6, 4, True)(x)
    assert recorder.calls == []

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


@pytest.mark.parametrize("kind", [fp8.Linear, models_f32.Linear])
def test_every_launch_is_on_the_inputs_device(monkeypatch, kind):
    """An input on cuda:1 while cuda:0 is the current device: the sampler and what reads its draws run on one device's stream, the input's."""
    current, seen = [0], []

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *error):
            current[0] = self.before

    class Library:
        def __getattr__(self, name):
            def entry(*args):
                seen.append((name, current[0]))
                return 0
            return entry

    class Tensor:
        """A tensor as far as the layers look at it, on cuda:1."""
        device, is_cuda, requires_grad, dtype = torch.device("cuda", 1), True, False, torch.float32

        def __init__(self, *shape):
            self.shape = torch.Size(shape)

        def data_ptr(self):
            return 4096

        def numel(self):
            return self.shape.numel()

        def view(self, *shape):
            return Tensor(*shape)

        def contiguous(self):
            return self

        def __getitem__(self, i):
            return Tensor(*self.shape[1:])

    monkeypatch.setattr(_lib, "lib", lambda: Library())
    monkeypatch.setattr(_lib, "current_stream", lambda: None)
    monkeypatch.setattr(torch.cuda, "device", Device)
    # the cast and the product decide by their tensors (fp8._launch)
    monkeypatch.setattr(fp8, "quantize_fp8", lambda w, rows: seen.append(("cast", w.device.index)) or w)
    monkeypatch.setattr(fp8, "linear_fp8", lambda x, w, *a, **kw: seen.append(("product", x.device.index)) or w)
    m = kind(6, 4, True)
    monkeypatch.setattr(torch, "empty", lambda shape, **kw: Tensor(*shape))
    m._sigma, m._mu_dev, m._bias_dev = Tensor(4, 6), Tensor(4, 6), Tensor(4)
    with q.mc_context(3, 1):
        m(Tensor(1, 2, 6))
    assert len(seen) >= 2 and seen[0][0] == "qbnn_sample_weights_f32" and {device for _, device in seen} == {1}


@pytest.mark.parametrize("kind", [fp8.Linear, models_f32.Linear])
def test_noise_for_fewer_samples_is_refused(recorder, kind):
    """eps is read [samples, out_features * in_features]: one that is shorter would be read past its end."""
    m = kind(6, 4, True)
    with q.mc_context(3, 1):
        for eps in (torch.zeros(24), torch.zeros(2, 24), torch.zeros(3, 23)):
            with pytest.raises(ValueError, match="eps"):
                m(torch.zeros(1, 2, 6), eps=eps)
    assert recorder.calls == []

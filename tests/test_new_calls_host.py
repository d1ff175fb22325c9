"""The host side of rotary positions, shared prefixes and adapters, on the CPU: which GPU a
call runs on, and that nothing goes by an address."""
import contextlib

import pytest


class Elsewhere:
    """Tensors of GPU 1 while GPU 0 is the current one, as far as the checks before a call go."""

    def __init__(self, monkeypatch, pk):
        import torch

        self.current, self.entered = 0, []

        @contextlib.contextmanager
        def device(index):
            self.entered.append(index)
            before, self.current = self.current, index
            try:
                yield
            finally:
                self.current = before

        monkeypatch.setattr(pk, "_current_device", lambda: self.current)
        monkeypatch.setattr(torch.cuda, "device", device)


@pytest.fixture
def pk():
    from cudalm_w4a16 import paged_kv

    return paged_kv


def test_the_current_gpu_is_asked_for_at_every_call(monkeypatch, pk):
    seen = iter([0, 1, 1])
    monkeypatch.setattr(pk, "_current_device", lambda: next(seen))
    assert pk._elsewhere(1) and not pk._elsewhere(1) and pk._elsewhere(0)
    assert not pk._elsewhere(-1)  # (tensors of the CPU are refused by the checks)


def test_calls_run_on_the_gpu_of_their_tensors(monkeypatch, pk):
    """The launch, and the memory for the result, come after the change of device."""
    import torch

    from cudalm_w4a16 import lora, rotary

    else_ = Elsewhere(monkeypatch, pk)

    class Tensor:
        def __init__(self, *shape, dtype=torch.bfloat16):
            self.t = torch.empty(*shape, dtype=dtype)

        def __getattr__(self, name):
            return getattr(self.t, name)

        def get_device(self):
            return 1

    class Stop(Exception):
        pass

    def reached(*a, **k):
        assert else_.current == 1, "on another GPU"
        raise Stop

    monkeypatch.setattr(rotary, "_empty", reached)
    rot = rotary.Rotary.__new__(rotary.Rotary)
    rot.index, rot.axes, rot.pairs, rot._bytes = 1, 1, 8, b""
    with pytest.raises(Stop):
        rotary.rotate(Tensor(3, 2, 16), Tensor(3, dtype=torch.int32), rot)
    monkeypatch.setattr(lora, "_empty", reached)
    with pytest.raises(Stop):
        lora.plan(Tensor(5, dtype=torch.int32), 3)
    monkeypatch.setattr(lora, "_stream", reached)
    plan = lora.Plan.__new__(lora.Plan)
    plan.M, plan.adapters, plan.index, plan.at = 5, 3, 1, 0
    with pytest.raises(Stop):
        lora.add(Tensor(5, 16), [Tensor(5, 8)], [Tensor(3, 8, 16)], [Tensor(3, 8, 8)], plan)
    monkeypatch.setattr(pk, "_out_like", reached)
    k, v = Tensor(4, 2, 16, 64), Tensor(4, 2, 2, 64, 8)
    int32 = lambda *s: Tensor(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(Stop):
        pk.decode_shared(Tensor(3, 4, 64), k, v, int32(3, 2), int32(3), int32(2), int32(1))
    with pytest.raises(Stop):
        rotary.append(Tensor(3, 4, 64), Tensor(3, 2, 64), Tensor(3, 2, 64), k, v, int32(3, 2), int32(3), rot)
    assert else_.entered == [1] * 5 and else_.current == 0


@pytest.mark.parametrize("value", [2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1])
@pytest.mark.parametrize("name", ["window", "sinks", "max_len", "max_shared"])
def test_options_past_32_bits_are_refused(monkeypatch, pk, name, value):
    import torch

    class Tensor:
        def __init__(self, *shape, dtype=torch.bfloat16):
            self.t = torch.empty(*shape, dtype=dtype)

        def __getattr__(self, attr):
            return getattr(self.t, attr)

        def get_device(self):
            return 0

    monkeypatch.setattr(pk, "_current_device", lambda: 0)
    int32 = lambda *s: Tensor(*s, dtype=torch.int32)  # noqa: E731
    q = Tensor(3, 4, 64)
    with pytest.raises(ValueError, match=name):
        pk.decode_shared(q, Tensor(4, 2, 16, 64), Tensor(4, 2, 2, 64, 8), int32(3, 2), int32(3), int32(2), int32(1), out=q,
                         **{name: value})

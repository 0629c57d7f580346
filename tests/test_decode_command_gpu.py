"""The command `python -m l2domain_b200.decode` on the GPU."""
import json

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from l2domain_b200 import decode  # noqa: E402


def run(monkeypatch, capsys, *args):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    monkeypatch.setattr("sys.argv", ["decode", "--batch", "2", "--length", "100", "--hidden", "256", "--heads", "4", "--kv-heads", "2",
                                     "--head-dim", "64", *args])
    assert decode.main() == 0
    return json.loads(capsys.readouterr().out)


def test_first_step_waits_for_its_inputs(monkeypatch, capsys):
    """The stream that fills the cache and the positions is kept busy, and free memory holds positions out of range: a
    step that does not wait reads those, and the status says so."""
    run(monkeypatch, capsys, "--steps", "5")  # once before, since loading a kernel waits for the device

    class Late(decode.DecodeAttention):
        def __init__(self, *a, **kw):
            super().__init__(*a, **kw)
            junk = [torch.full((128,), 0x7f7f7f7f, dtype=torch.int32, device="cuda") + 0 for _ in range(16384)]
            del junk
            torch.cuda.synchronize()
            torch.cuda._sleep(2_000_000_000)

    monkeypatch.setattr(decode, "DecodeAttention", Late)
    assert run(monkeypatch, capsys, "--steps", "5")["status"] == 0


def test_bytes_are_those_of_the_timed_steps(monkeypatch, capsys):
    """Ten steps before the timed ones, and every step, make the cache a token longer."""
    got = run(monkeypatch, capsys, "--steps", "7")
    keys = sum(100 + 10 + i for i in range(7)) / 7
    assert got["cache_bytes"] == 2 * 2 * keys * 2 * 64 * 2

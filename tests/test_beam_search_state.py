"""BeamSearch's own state and the objects' sizes, without a GPU."""
import pytest
import torch

from tabby_amd import beam
from tabby_amd import sampler as S


def _search(groups=3, beams=2):
    run = beam.BeamSearch(groups, beams, 50, 4, end_ids=(9,), device="cpu")
    run.length = 3
    run.tokens[::beams] = torch.tensor([[1, 2, 3, 0], [4, 9, 0, 0], [5, 6, 7, 0]], dtype=torch.int32)[:groups]
    run.scores[:, 0] = torch.tensor([-1.0, -2.0, -3.0])[:groups]
    return run


@pytest.mark.parametrize("code,text", [(S.TABBY_EEMPTY, "no continuation"), (S.TABBY_EDOMAIN, "NaN")])
def test_the_other_groups_results_when_one_failed(code, text):
    run = _search()
    assert run.best() == [([1, 2, 3], -1.0), ([4, 9], -2.0), ([5, 6, 7], -3.0)] == run.best(strict=False)
    run.status[1] = code
    with pytest.raises(S.SamplingError, match=f"group 1: .*{text}"):
        run.best()
    assert run.best(strict=False) == [([1, 2, 3], -1.0), None, ([5, 6, 7], -3.0)]


def test_a_step_is_not_captured(monkeypatch):
    # A replay would read the scores of the step that was captured and write its tokens into the same column again.
    import contextlib
    run = _search()
    monkeypatch.setattr(beam, "call_on", lambda device, stream: (contextlib.nullcontext(), 0))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ValueError, match="captured"):
        run.step(torch.zeros(6, 50))
    assert run.length == 3


def test_sizes_past_32_bits_are_refused():
    # The C entries take 32-bit sizes: what does not fit would be taken modulo 2^32.
    from tabby_amd import mx4
    for rows, cols in ((2 ** 32 + 1, 5), (5, 2 ** 32 + 1), (2 ** 31, 1)):
        with pytest.raises(ValueError, match="32 bits"):
            mx4.Mx4Matrix(rows, cols, device="cpu")
    for sizes in ({"vocab_max": 2 ** 32 + 100}, {"vocab_max": 100, "groups_max": 2 ** 32 + 1},
                  {"vocab_max": 100, "beams_max": 2 ** 32 + 4}, {"vocab_max": 100, "count_max": 2 ** 32 + 8}):
        with pytest.raises(ValueError, match="32 bits"):
            beam.BeamSelect(**sizes, device="cpu")

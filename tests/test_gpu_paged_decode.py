"""The example of serving with a paged cache: prompt, forks, captured decode
steps, a freed sequence, compaction, more steps; every sequence's last result
is what its whole history gives as one prompt of its own."""
import importlib.util
import pathlib

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

PATH = pathlib.Path(__file__).resolve().parents[1] / "llama.zig_amd" / "examples" / "paged_decode.py"


def _example():
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_steps_equal_a_prompt_of_the_whole_history(window, sinks):
    m = _example()
    server, seen, last = m.main(prompt_tokens=75, steps=20, window=window, sinks=sinks)
    assert [server.lens[q] for q in (0, 1, 2)] == [115, 0, 115]
    assert {q: x.shape[0] for q, x in seen.items()} == {0: 115, 1: 95, 2: 115}
    # no page is in two lists, none is lost
    assert len(server.free) + len(server.used) == server.caches[0].n_pages
    assert sorted(server.used) == list(range(len(server.used)))
    for q in (0, 2):
        whole = m.Server(window=window, sinks=sinks)
        want = whole.prompt(0, seen[q]).double()
        # Activations are quantized to 8 bits before each of the four products (a step and a prompt sum them in
        # another order, and a code at a tie may fall to its other side: 2^-8 of a block's largest value in one
        # of thousands), keys and values are rounded to 11 bits: far under 1 % of the result.
        assert float((last[q].double() - want).norm() / want.norm()) < 1e-2
    assert not torch.equal(last[0], last[2])

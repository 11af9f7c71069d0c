"""What DecodeModel checks on the host before it launches anything (no GPU needed)."""
import pytest

from rqmv.decode import DecodeModel


class Launches:
    """Stands for a captured step."""

    def __init__(self, sampling=None):
        self.count, self.sampling = 0, sampling

    def launch(self, stream):
        self.count += 1


class Settings:
    def __init__(self, draws):
        self.draws = lambda: draws


@pytest.fixture
def model():
    m = DecodeModel.__new__(DecodeModel)  # (its host state alone)
    m.max_ctx, m._pos = 32, 8
    return m


def test_several_replays_do_not_share_a_random_number(model):
    graph = Launches(Settings(True))
    with pytest.raises(ValueError, match="one random number"):
        model.replay(graph, None, 2)
    assert graph.count == 0 and model._pos == 8
    model.replay(graph, None)
    assert graph.count == 1 and model._pos == 9


@pytest.mark.parametrize("sampling", [None, Settings(False)])
def test_several_replays_without_a_random_number(model, sampling):
    graph = Launches(sampling)
    model.replay(graph, None, 5)
    assert graph.count == 5 and model._pos == 13
    with pytest.raises(ValueError, match="run past the cache"):
        model.replay(graph, None, 20)
    plain = Launches()
    del plain.sampling  # a graph that capture() did not make
    model.replay(plain, None, 2)
    assert plain.count == 2

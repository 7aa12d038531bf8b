"""Captures beside a model that holds captured graphs of its own: MapAnything captures its forwards under inference mode,
callers capture the streaming operators in whichever mode they run in, before or after."""

import pytest
import torch

from tests_helpers import CASES, make_views, released_config

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def loaded():
    from mapanything.models import MapAnything

    return MapAnything(**released_config()).load_synthetic_weights().to("cuda").eval()


@pytest.fixture()
def model(loaded):
    loaded._graphs.clear()
    yield loaded
    loaded._graphs.clear()


@pytest.fixture()
def views():
    return make_views(CASES["cfg1_224"])


def _infer(model, views):
    out = model.infer(views, use_amp=True, apply_mask=False)
    assert len(model._graphs) > 0  # the model holds a graph
    return [v["pts3d"].clone() for v in out]


def _randn(*shape, seed, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


class Calls:
    """The streaming operators over one scene; `run` makes every call of them and returns what they gave."""

    def __init__(self, grad=True):
        from mapanything.kv_cache import KVBatch, PagedKVCache
        from uniception.models.libs.croco.pos_embed import RoPEAxes

        def ints(x):
            return torch.tensor(x, dtype=torch.int32, device="cuda")

        self.cache = PagedKVCache(8, 16, 2, torch.bfloat16)
        self.cache.k.zero_()
        self.cache.v.zero_()
        self.batch = KVBatch(ints([[5, 1, 3]]), ints([40]), ints([0, 9]), max_new=9, max_kv=40)
        self.rows = ints([0, 40])
        self.x = [_randn(9, 2, 64, seed=i) for i in range(3)]
        self.pos = torch.randint(0, 50, (9, 3), generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
        self.rope = RoPEAxes((8, 12, 12), freq=100.0)
        self.leaf = _randn(1, 2, 9, 64, seed=7).requires_grad_() if grad else None

    def run(self, leaf=None):
        q, k, v = self.x
        out = []
        with torch.no_grad():
            k = self.rope(k.transpose(0, 1)[None], self.pos)[0].transpose(0, 1)
            self.cache.write(k, v, self.batch)
            out += self.cache.read(self.batch, self.rows, 40)
            out.append(self.cache.attend(q, self.batch, mask_block=1))
        if leaf is not None:
            y = self.rope(leaf, self.pos)
            out += [y.detach(), *torch.autograd.grad(y, leaf, torch.ones_like(y))]
        return out

    def capture_and_check(self):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.run(self.leaf)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = self.run(self.leaf)
        return graph, got

    def replay_and_check(self, graph, got, turn):
        with torch.no_grad():
            for i, x in enumerate(self.x):
                x.copy_(_randn(*x.shape, seed=100 + 10 * turn + i))
            self.pos.add_(3)
            if self.leaf is not None:
                self.leaf.copy_(_randn(*self.leaf.shape, seed=200 + turn))
        graph.replay()
        torch.cuda.synchronize()
        got = [g.clone() for g in got]
        want = self.run(None if self.leaf is None else self.leaf.detach().clone().requires_grad_())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_capture_outside_inference_mode_beside_a_model(model, views):
    """infer, keep the model (and its graph), capture every streaming operator outside inference mode, replay both in
    turn: the model's graphs leave nothing behind that a later capture meets."""
    first = _infer(model, views)
    calls = Calls()
    graph, got = calls.capture_and_check()
    for turn in range(3):
        calls.replay_and_check(graph, got, turn)
        assert all(torch.equal(a, b) for a, b in zip(first, _infer(model, views)))
    model._graphs.clear()  # captured again while the caller's graph lives
    assert all(torch.equal(a, b) for a, b in zip(first, _infer(model, views)))
    calls.replay_and_check(graph, got, 7)


def test_model_captures_beside_a_callers_inference_mode_graph(model, views):
    """The other order: a caller's graph, captured under inference mode and kept, does not stop the model's capture."""
    with torch.inference_mode():
        calls = Calls(grad=False)
        graph, got = calls.capture_and_check()
        calls.replay_and_check(graph, got, 0)
    first = _infer(model, views)
    with torch.inference_mode():
        calls.replay_and_check(graph, got, 1)
    assert all(torch.equal(a, b) for a, b in zip(first, _infer(model, views)))


def test_model_capture_leaves_the_random_generator_alone(model, views):
    """Random numbers drawn after infer() (its capture, its replays) are those that would be drawn without it."""
    torch.manual_seed(5)
    want = [torch.randn(1000, device="cuda") for _ in range(3)]
    torch.manual_seed(5)
    got = []
    for _ in range(3):
        got.append(torch.randn(1000, device="cuda"))
        _infer(model, views)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

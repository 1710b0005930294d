"""``moe.run``'s scratch: one set a stream, a thread and a capture (host logic without a GPU), and on the GPU calls on
two streams and replays of two graphs beside one another with the bits of calls in a row."""

import threading

import pytest
import torch

BF = torch.bfloat16


def routed(device, kind="16-bit", experts=6, dims=128, width=64, seed=1):
    from tensorfold_b200 import experts as grouped
    from tensorfold_b200 import experts16, moe

    if device == "cpu":
        ex = experts16.Experts16(torch.zeros((experts, 2 * width, dims), dtype=BF), torch.zeros((experts, dims, width), dtype=BF),
                                 width, dims, True)
        return moe.Routed(torch.zeros((experts, dims), dtype=BF), ex, 2, shared=False)
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return (torch.randn(shape, generator=g, device=device) * 0.1).to(BF)

    if kind == "16-bit":
        ex = experts16.make([normal(experts, width, dims), normal(experts, width, dims)], normal(experts, dims, width))
    else:
        def mlx(n, k):
            words = torch.randint(-2 ** 31, 2 ** 31, (experts, n, k // 8), generator=g, device=device, dtype=torch.int64).to(torch.int32)
            return words, normal(experts, n, k // 64).abs() * 0.1, normal(experts, n, k // 64)

        ex = grouped.make([mlx(width, dims), mlx(width, dims)], mlx(dims, width), 64)
    return moe.Routed(normal(experts, dims), ex, 2, shared=False)


@pytest.fixture
def calls(monkeypatch):
    """``moe.run`` without its launches: what it would have run on, by the stream and the capture that the test names."""

    from tensorfold_b200 import _lib, moe

    state = {"stream": 1, "capture": 0, "used": []}
    monkeypatch.setattr(moe, "_scratch", {})
    monkeypatch.setattr(_lib, "stream", lambda device: state["stream"])
    monkeypatch.setattr(_lib, "capture", lambda stream: state["capture"], raising=False)
    monkeypatch.setattr(moe, "layer", lambda x, m, buf, out: state["used"].append(buf))
    layer = routed("cpu")

    def call(stream=1, capture=0, rows=5, prefill=False):
        state.update(stream=stream, capture=capture)
        moe.run(torch.zeros((rows, 128), dtype=BF), layer, prefill=prefill)
        return state["used"][-1]

    return call


def test_a_stream_keeps_its_scratch_and_shares_it_with_no_other(calls):
    one, two = calls(stream=1), calls(stream=2)
    assert one is not two and calls(stream=1) is one and calls(stream=2) is two
    assert calls(stream=1, rows=16) is one and calls(stream=1, rows=17) is not one and calls(stream=1, prefill=True) is not one
    assert one.y.data_ptr() != two.y.data_ptr() and one.plan.items.data_ptr() != two.plan.items.data_ptr()


def test_threads_do_not_share_scratch(calls):
    mine, other = calls(), []
    t = threading.Thread(target=lambda: other.append(calls()))
    t.start()
    t.join()
    assert other[0] is not mine and calls() is mine


def test_a_capture_has_scratch_of_its_own(calls):
    """Shared by the capture's calls on one stream, with no other capture and no eager call; the last capture's is let go
    for the next one's."""

    from tensorfold_b200 import moe

    eager, first = calls(), calls(capture=7)
    assert first is not eager and calls(capture=7) is first and calls(stream=2, capture=7) not in (first, eager)
    second = calls(capture=8)
    assert second not in (first, eager) and calls() is eager and calls(capture=8) is second
    assert [sorted(who[1] for who in kept) for kept in moe._scratch.values()] == [[0, 8]]


def test_scratch_is_bounded(calls):
    from tensorfold_b200 import moe

    made = [calls(stream=s) for s in range(1, 40)]
    assert [len(kept) for kept in moe._scratch.values()] == [moe.SCRATCH_KEPT]
    assert calls(stream=39) is made[-1] and calls(stream=1) is not made[0]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["16-bit", "4-bit"])
def test_two_streams_run_layers_of_one_shape(kind):
    """Calls enqueued in turn on two streams without waiting: the bits of the same calls in a row."""

    from tensorfold_b200 import moe

    layers = [routed("cuda", kind, 6, 512, 256, seed) for seed in (1, 2)]
    g = torch.Generator(device="cuda").manual_seed(3)
    xs = [(torch.randn((rows, 512), generator=g, device="cuda") * 0.5).to(BF) for rows in (190, 130)]
    want = [moe.run(x, layer) for x, layer in zip(xs, layers)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(moe.run(xs[k], layers[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(y, want[k]) for y in got[k])


@pytest.mark.gpu
def test_captures_are_told_apart():
    from tensorfold_b200 import _lib

    s, dev, seen = torch.cuda.Stream(), torch.device("cuda", 0), []
    torch.cuda.synchronize()
    for _ in range(2):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            seen += [_lib.capture(_lib.stream(dev)), _lib.capture(_lib.stream(dev))]
            torch.zeros((4,), device="cuda")
    assert seen[0] == seen[1] != seen[2] == seen[3] and 0 not in seen
    with torch.cuda.stream(s):
        assert _lib.capture(_lib.stream(dev)) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["16-bit", "4-bit"])
def test_graphs_of_run_replay_beside_one_another(kind):
    """Two captured calls of one shape, replayed on two streams beside an eager call on a third."""

    from tensorfold_b200 import moe

    layer = routed("cuda", kind, 6, 512, 256)
    g = torch.Generator(device="cuda").manual_seed(4)
    xs = [(torch.randn((150, 512), generator=g, device="cuda") * 0.5).to(BF) for _ in range(3)]
    want = [moe.run(x, layer) for x in xs]
    streams, held = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for k in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = moe.run(xs[k], layer)
        held.append((graph, out))
    torch.cuda.synchronize()
    for _ in range(20):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                held[k][0].replay()
        again = moe.run(xs[2], layer)
        torch.cuda.synchronize()
        assert torch.equal(held[0][1], want[0]) and torch.equal(held[1][1], want[1]) and torch.equal(again, want[2])

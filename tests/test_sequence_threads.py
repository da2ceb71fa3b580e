"""The list of living autograd graphs, by which a captured backward pass is refused in time, with several threads at work on it."""
import threading

import torch

from dm_amd.neural_nets import sequence
from dm_amd.runtime import hip


class Node:
    next_functions = ()


def test_a_graph_noted_during_a_sweep_is_kept(monkeypatch):
    """one thread sweeps dead entries out; another notes a graph just before the swept list is put in place"""
    monkeypatch.setattr(hip, "stream", lambda *a: 0)
    late, threads = Node(), []

    class Slow(list):
        def __setitem__(self, at, value):
            t = threading.Thread(target=sequence._note_graph, args=(late, torch.zeros(1)))
            threads.append(t)
            t.start()
            t.join(0.3)                                        # (it either gets through, or waits for the sweep to end)
            super().__setitem__(at, value)

    graphs = Slow([lambda: None] * 4095)
    monkeypatch.setattr(sequence, "_graphs", graphs)
    monkeypatch.setattr(sequence, "_sweep_at", 4096)
    first = Node()
    sequence._note_graph(first, torch.zeros(1))
    assert len(threads) == 1
    threads[0].join(10)
    assert not threads[0].is_alive() and {r() for r in graphs} == {first, late}


def test_the_stream_is_that_of_the_inputs_device(monkeypatch):
    """inputs on the second device, whose current stream is the default one, while the first device is current and on another stream: the graph belongs to
    the default stream"""
    class OnSecond:
        device = torch.device("cuda", 1)
        requires_grad = is_leaf = True
        get_device = staticmethod(lambda: 1)

    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", {0: 77, 1: 0}.__getitem__, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(sequence, "_graphs", [])
    node = Node()
    sequence._note_graph(node, OnSecond())
    assert node.stream == 0 and [r() for r in sequence._graphs] == [node]


def test_many_living_graphs_are_not_swept_at_every_call(monkeypatch):
    """with thousands of graphs alive, a sweep frees nothing: the next one waits until the list has doubled"""
    monkeypatch.setattr(hip, "stream", lambda *a: 0)
    looks, alive = [0], [Node() for _ in range(12000)]

    class Counted(list):
        def __setitem__(self, at, value):
            looks[0] += 1
            super().__setitem__(at, value)

    monkeypatch.setattr(sequence, "_graphs", Counted())
    monkeypatch.setattr(sequence, "_sweep_at", 4096)
    x = torch.zeros(1)
    for node in alive:
        sequence._note_graph(node, x)
    assert [r() for r in sequence._graphs] == alive and looks[0] <= 3
    del alive[6000:], node
    for _ in range(30000):                                     # dead ones are swept out all the same
        sequence._note_graph(Node(), x)
    assert len(sequence._graphs) < 30000 and [r() for r in sequence._graphs[:6000]] == alive

"""Workspaces that captured graphs use (nanovllm_b200.fp8_attention.workspace): every graph has its own, zero
before the first replay, outside the graph's memory pool, and for good; and a recorded error stays."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)


def _case(seqs, longest, seed):
    from nanovllm_b200 import workloads
    return workloads.decode_case(seqs, 32, 8, 1, longest, seed=seed, device="cuda", block_size=64)


def _decode(c):
    from nanovllm_b200 import fp8_decode_attention
    return fp8_decode_attention(c.q, c.k_cache, c.v_cache, c.block_tables, c.context_lens, c.scale)


def _capture(c, pool=None, work=None):
    """(graph, output, workspace) of one decode call, with work before and after it."""
    from nanovllm_b200 import fp8_attention
    before = set(fp8_attention._WORKSPACES)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, pool=pool):
        if work is not None:
            (work * 2).sum()
        out = _decode(c)
        if work is not None:
            (work * 3).sum()
    new = [k for k in fp8_attention._WORKSPACES if k not in before]
    assert len(new) == 1
    return g, out, fp8_attention._WORKSPACES[new[0]]


def test_each_graph_has_a_workspace_of_zeros():
    """Small, large, small again, all of one pool, among other memory of that pool; replayed in the
    order that never runs the first one first."""
    cases = [_case(4, 900, 1), _case(64, 3000, 2), _case(7, 500, 3)]
    want = [_decode(c) for c in cases]
    junk = torch.full((1 << 22,), 3.0, device="cuda")
    graphs, pool = [], None
    for c in cases:
        graphs.append(_capture(c, pool, junk))
        pool = graphs[0][0].pool()
    assert len({ws.data_ptr() for _, _, ws in graphs}) == 3
    for _, _, ws in graphs:
        assert not bool(ws.any())                       # before any replay
    for i in (2, 1, 0, 1, 2, 0):
        graphs[i][1].zero_()
        graphs[i][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[i][1], want[i])
    for _, _, ws in graphs:
        assert not bool(ws[:256].any())                 # counters and error word


def test_graphs_replayed_at_once():
    cases = [_case(16, 2000, 4), _case(16, 2000, 5)]
    want = [_decode(c) for c in cases]
    graphs = [_capture(c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, out, _), w in zip(graphs, want):
        assert torch.equal(out, w)


def test_a_larger_call_in_the_same_capture():
    """The first launch keeps its workspace when a later one of the same capture needs more."""
    a, b = _case(2, 300, 6), _case(64, 3000, 7)
    want = _decode(a), _decode(b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out_a = _decode(a)
        out_b = _decode(b)
        junk = torch.full((1 << 20,), 7.0, device="cuda")
    for _ in range(3):
        out_a.zero_(), out_b.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out_a, want[0]) and torch.equal(out_b, want[1])
    assert bool((junk == 7).all())


def test_a_capture_on_a_stream_with_a_workspace():
    """A stream's workspace is not the captures' on it, nor theirs the stream's."""
    from nanovllm_b200 import fp8_attention
    c = _case(8, 1500, 8)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        want = _decode(c)
        mine = fp8_attention.workspace(DEVICE, 0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = _decode(c)
        theirs = fp8_attention.workspace(DEVICE, 0)
    assert mine.data_ptr() != theirs.data_ptr()
    g.replay()
    with torch.cuda.stream(s):
        again = _decode(c)
        assert fp8_attention.workspace(DEVICE, 0) is mine
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(again, want)


def test_an_error_of_a_graph_stays_through_its_replays():
    from nanovllm_b200 import fp8_attention
    assert fp8_attention.device_error(DEVICE) == 0
    g, _, ws = _capture(_case(4, 400, 9))
    word = ws[:4].view(torch.int32)
    word.fill_(1)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert fp8_attention.device_error(DEVICE) == 1 and fp8_attention.device_error() == 1
    word.zero_()
    assert fp8_attention.device_error() == 0


def test_an_error_outlives_a_replaced_workspace():
    from nanovllm_b200 import fp8_attention
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ws = fp8_attention.workspace(DEVICE, 100)
        ws[:4].view(torch.int32).fill_(2)
        ws[4:].fill_(0xEE)
        larger = fp8_attention.workspace(DEVICE, ws.numel() + 1)
        torch.cuda.synchronize()
        assert larger.numel() > ws.numel() and not bool(larger[4:].any())
        assert fp8_attention.device_error(DEVICE) == 2
        larger[:4].zero_()
    torch.cuda.synchronize()
    assert fp8_attention.device_error(DEVICE) == 0


def test_first_call_of_a_process_inside_a_capture():
    """Nothing has run before: the workspace's stream and memory are made during the capture."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = (
        "import sys; sys.path[:0] = ['.', 'my-nano-vllm_b200']\n"
        "import torch\n"
        "from nanovllm_b200 import fp8_attention, fp8_decode_attention, workloads\n"
        "c = workloads.decode_case(5, 32, 8, 1, 700, seed=1, device='cuda', block_size=64)\n"
        "call = lambda: fp8_decode_attention(c.q, c.k_cache, c.v_cache, c.block_tables, c.context_lens, c.scale)\n"
        "torch.cuda.synchronize()\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    out = call()\n"
        "for _ in range(3):\n"
        "    out.zero_(); g.replay(); torch.cuda.synchronize()\n"
        "    got = out.clone()\n"
        "assert torch.equal(got, call())\n"
        "assert fp8_attention.device_error() == 0\n"
        "print('captured first')\n")
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured first" in run.stdout, run.stderr[-2000:]

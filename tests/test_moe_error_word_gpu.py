"""The error word of fp8_moe: what a wait that gave up recorded stays until it is read, whatever the
workspaces of the stream do and however often a captured graph is replayed.  The recording is made by the
wait's diagnostics entry point, with no word of its own, as fp8_moe's launches have none."""
import os
import subprocess
import sys

import pytest
import torch

from test_moe_gpu import _inputs, _run

pytestmark = pytest.mark.gpu


def _read(clear=0):
    from nanovllm_b200 import _lib
    word = torch.full((1,), -1, dtype=torch.int32, device="cuda")
    _lib.check(_lib.lib.fp8attn_fp8_moe_read_error(word.data_ptr(), clear,
                                                   torch.cuda.current_stream().cuda_stream))
    return int(word)


def _record():
    """A wait on counters that stay below the value, for 1 us."""
    from nanovllm_b200 import _lib
    zeros = torch.zeros(32, dtype=torch.int32, device="cuda")
    reached = torch.empty_like(zeros)
    _lib.check(_lib.lib.fp8attn_diag_counter_wait(zeros.data_ptr(), 1, 1000, reached.data_ptr(), 0,
                                                  torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert not bool(reached.any())


@pytest.fixture(autouse=True)
def _clean():
    from nanovllm_b200 import fp8_attention
    torch.cuda.synchronize()
    assert fp8_attention.device_error() == 0
    yield
    torch.cuda.synchronize()
    _read(clear=1)
    assert fp8_attention.device_error() == 0


def test_survives_larger_workspaces():
    from nanovllm_b200 import fp8_attention
    device = torch.device("cuda", torch.cuda.current_device())
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        a = _inputs(3, 256, 128, 8, 1)
        _run(a, 2)
        _record()
        assert fp8_attention.device_error(device) == 1
        for nbytes in (1 << 17, 1 << 20):
            fp8_attention.workspace(device, nbytes)
            assert fp8_attention.device_error(device) == 1 and fp8_attention.device_error() == 1
        _run(a, 2)
        assert _read(clear=1) == 1 and _read() == 0
        assert fp8_attention.device_error(device) == 0


def test_survives_replays():
    from nanovllm_b200 import fp8_attention
    a = _inputs(5, 512, 256, 16, 2)
    want = _run(a, 4)
    graphs = []
    for _ in range(2):                                  # two graphs of one capture stream
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _run(a, 4)
        graphs.append((g, out))
    _record()
    for g, out in graphs * 2:
        g.replay()
        torch.cuda.synchronize()
        assert fp8_attention.device_error() == 1
        for p, q in zip(want, out):
            assert torch.equal(p, q)


def test_first_call_of_a_process_inside_a_capture():
    """Nothing of the library has run before: the word needs no preparation."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = (
        "import sys; sys.path[:0] = ['tests', '.', 'my-nano-vllm_b200']\n"
        "import torch\n"
        "from nanovllm_b200 import fp8_attention, fp8_ffn\n"
        "gen = torch.Generator(device='cuda').manual_seed(1)\n"
        "r = lambda *s: torch.randn(*s, generator=gen, device='cuda')\n"
        "e = lambda *s: r(*s).to(torch.float8_e4m3fn)\n"
        "o = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device='cuda')\n"
        "a = (r(4, 256).bfloat16(), e(4, 256), o(4, 2), r(8, 256).bfloat16(), e(8, 256, 256), o(8, 2, 2),\n"
        "     e(8, 256, 128), o(8, 2, 1), 2)\n"
        "torch.cuda.synchronize()\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    out = fp8_ffn.fp8_moe(*a)\n"
        "for _ in range(3):\n"
        "    out.zero_(); g.replay(); torch.cuda.synchronize()\n"
        "    got = out.clone()\n"
        "assert torch.equal(got, fp8_ffn.fp8_moe(*a))\n"
        "assert fp8_attention.device_error() == 0\n"
        "print('captured first')\n")
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured first" in run.stdout, run.stderr[-2000:]


def test_a_call_s_own_word_is_used_where_it_brings_one():
    from nanovllm_b200 import _lib
    zeros = torch.zeros(32, dtype=torch.int32, device="cuda")
    reached, word = torch.empty_like(zeros), torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.check(_lib.lib.fp8attn_diag_counter_wait(zeros.data_ptr(), 1, 1000, reached.data_ptr(),
                                                  word.data_ptr(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert int(word) == 1 and _read() == 0
    assert _lib.lib.fp8attn_fp8_moe_read_error(None, 0, None) == _lib.EINVAL

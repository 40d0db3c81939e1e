"""GPU: the capture window of this package (ops.capture) against Python's cyclic garbage collector -- the crash mechanism found behind
GPUTEST_r04 (profiles/r05_capture_crash.txt): an OLD CUDAGraph kept alive only by a reference cycle is
finalised by whatever allocation triggers the collector; inside a capture window its destructor (hipDeviceSynchronize on ROCm) kills the
process.  Each scenario runs in a subprocess so that a regression is an assertion, not a dead test session."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_SCRIPT = r'''
import gc, sys
sys.path.insert(0, %(root)r)
import torch
from multiagentperception_amd import ops

def old_graph_garbage():
    x = torch.zeros(1 << 18, device="cuda")
    s = torch.cuda.Stream(); s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 2 + 1
    torch.cuda.current_stream().wait_stream(s); torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        y = x * 2 + 1
    g.replay(); torch.cuda.synchronize()
    cyc = [g, x, y]; cyc.append(cyc)          # only the cyclic collector can free this

mode = sys.argv[1]
x2 = torch.zeros(1 << 18, device="cuda")
if mode == "guarded":
    gc.collect(); gc.set_threshold(1, 1, 1)   # the collector runs at (nearly) every allocation from here on
    old_graph_garbage()
    was = gc.isenabled()
    with ops.capture() as g2:                 # collects BEFORE the window, holds the collector off INSIDE it
        assert not gc.isenabled()
        z = x2 * 3
        junk = [[i] for i in range(5000)]     # allocations that would trigger the collector
        z = z + 1
    assert gc.isenabled() == was
    g2.replay(); torch.cuda.synchronize()
    assert float(z[0]) == 1.0
    print("GUARDED_OK")
'''


def _run(mode):
    return subprocess.run([sys.executable, "-c", _SCRIPT % {"root": ROOT}, mode], capture_output=True, text=True, timeout=300)


def test_capture_window_holds_the_garbage_collector_off():
    r = _run("guarded")
    assert r.returncode == 0 and "GUARDED_OK" in r.stdout, (r.returncode, r.stdout[-2000:], r.stderr[-4000:])


@pytest.mark.skip(reason="made a GPU process abort on purpose (a CUDAGraph finalised inside a capture window); what it showed: profiles/r05_capture_crash.txt")
def test_the_hazard_is_real_without_the_guard():
    """The sequence of the test above through a bare torch.cuda.graph: SIGABRT from a check inside at::cuda::CUDAGraph::~CUDAGraph (torch 2.10 /
    ROCm 7).  Not run any more, and without a body that could."""


def test_no_capture_site_bypasses_the_guard():
    """every torch.cuda.graph( in the package is the one inside ops.capture (ops.record_program drives capture_begin / capture_end itself,
    under the same collector guard)"""
    import re
    pkg = os.path.join(ROOT, "multiagentperception_amd")
    hits = []
    for fn in sorted(os.listdir(pkg)) + [os.path.join("models", f) for f in sorted(os.listdir(os.path.join(pkg, "models")))]:
        if fn.endswith(".py"):
            for i, line in enumerate(open(os.path.join(pkg, fn)), 1):
                if re.search(r"torch\.cuda\.graph\(", line) and not line.lstrip().startswith(("#", '"', "'")):
                    hits.append((fn, i))
    assert hits and all(fn == "ops.py" for fn, _ in hits), hits


def _repro(queues, script, args):
    env = dict(os.environ)
    env.pop("GPU_MAX_HW_QUEUES", None)
    if queues is not None:
        env["GPU_MAX_HW_QUEUES"] = str(queues)
    try:
        return subprocess.run([sys.executable, os.path.join(ROOT, "tools", *script)] + list(args),
                              capture_output=True, text=True, timeout=400, env=env)
    except subprocess.TimeoutExpired as e:           # an out-of-bounds pointer may also wedge the launch instead of faulting
        return subprocess.CompletedProcess(e.cmd, -9, stdout=str(e.stdout or ""), stderr="timed out (treated as killed)")


def test_recorded_programs_survive_bursts_of_exec_destruction_at_the_runtimes_default_queue_count():
    """The crash of GPUTEST_r04 (profiles/r05_capture_crash.txt): hipGraphLaunch of a MULTI-BRANCH exec faulted inside the runtime when the
    exec's streams shared the launch stream's hardware queue; at the runtime's default of 4 hardware queues a burst of exec destructions makes
    the next execs' streams pile onto one queue.  Every graph the package launches is single-branch (ops.record_program).  tools/r06/program_burst.py is the same burst pattern on recorded programs (4 recordings per
    iteration, 3 dropped at once, replays from 3-7 long-lived streams: 160 iterations here, 2 400 replays) and on the product's own forwards (engines dropped in bursts), with
    NO queue-count variable in the environment."""
    r = _repro(None, script=("r06", "program_burst.py"), args=("160", "4"))
    assert r.returncode == 0 and "SURVIVED" in r.stdout, (r.returncode, r.stdout[-500:], r.stderr[-1500:])


def test_the_package_sets_no_runtime_environment_variables():
    env = dict(os.environ)
    for k in ("GPU_MAX_HW_QUEUES", "TORCH_FR_BUFFER_SIZE"):
        env.pop(k, None)
    code = ("import os, sys; sys.path.insert(0, %r); import multiagentperception_amd, ptsemseg.models, multiagentperception_amd.parallel; "
            "print('ENV', os.environ.get('GPU_MAX_HW_QUEUES'), os.environ.get('TORCH_FR_BUFFER_SIZE'))" % ROOT)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "ENV None None" in r.stdout, (r.stdout[-300:], r.stderr[-1500:])


@pytest.mark.skip(reason="made the runtime read out of bounds on purpose; what it showed: profiles/r05_capture_crash.txt")
def test_the_runtime_defect_is_real_for_multi_branch_graphs_at_the_default_queue_count():
    """Multi-branch graphs in pure torch at 4 hardware queues (the runtime's default): SIGSEGV inside libamdhip64's hipGraphLaunch within a few
    hundred launches.  Not run any more, and without a body that could."""


def test_recorded_program_equals_the_eager_run_and_consists_of_single_branch_graphs():
    """ops.record_program: the same function run under the eager lanes and replayed from its recorded program gives the same bits on new
    input data; the verbs cut it into the expected windows (one graph per window, event edges between them); replays on several streams
    and in several threads' worth of interleavings stay ordered by the edges."""
    import torch
    from multiagentperception_amd import ops
    dev = torch.device("cuda:0")
    x = torch.randn(1 << 20, device=dev)
    w = torch.randn(512, 512, device=dev)

    def fn():
        L = ops.lanes(dev)
        y = x * 2
        with L.on(1, after=(0,)):
            a = y + 1
            for _ in range(20):                     # something long on lane 1: the edges, not luck, must order the consumers
                a = (a.view(-1, 512) @ w).view(-1) * 1e-2 + y
            tok = L.mark()
            b = a * 3
        c = y - 1
        L.wait(tok)
        d = c + a
        L.join(1)
        return d + b

    want0 = fn().clone()
    prog = ops.record_program(dev, fn, warmup=1)
    assert prog.n_graphs == 6 and len(prog.side) == 1, (prog.n_graphs, [st[0] for st in prog.prog])
    assert [st[0] for st in prog.prog] == ["graph", "sync", "graph", "record", "graph", "graph", "wait", "graph", "sync", "graph"]
    assert torch.equal(prog.replay(), want0)
    for seed in range(3):
        x.copy_(torch.randn(1 << 20, device=dev))
        want = fn().clone()
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            got = prog.replay().clone()
        torch.cuda.current_stream(dev).wait_stream(s)
        assert torch.equal(got, want), seed


def test_a_nested_recording_is_refused_and_a_failed_recording_leaves_no_capture_open():
    import torch
    from multiagentperception_amd import ops
    dev = torch.device("cuda:0")
    x = torch.zeros(16, device=dev)

    def bad():
        y = x + 1
        raise ValueError("boom")

    with pytest.raises(ValueError):
        ops.record_program(dev, bad, warmup=0)
    assert not torch.cuda.is_current_stream_capturing()
    with pytest.raises(ops.W2CError):
        ops.record_program(dev, lambda: ops.record_program(dev, lambda: x + 1, warmup=0), warmup=0)
    prog = ops.record_program(dev, lambda: x + 2, warmup=0)                # and recording still works afterwards
    assert float(prog.replay()[0]) == 2.0


def test_caller_streams_are_distinct_streams_and_the_queue_probe_runs():
    """ops.caller_streams (round 6: streams for a loop that keeps several engines in flight, picked so that they share no hardware queue
    with each other or with the value lane -- bench.py's forwards_in_flight) returns n distinct streams; ops.streams_share_queue answers
    True for a stream and itself and a bool for any pair.  (Which pairs share is the runtime's draw: profiles/r06_stream_queues.txt.)"""
    import torch
    from multiagentperception_amd import ops
    dev = torch.device("cuda:0")
    ss = ops.caller_streams(dev, 3)
    assert len(ss) == 3 and len({s.cuda_stream for s in ss}) == 3 and all(isinstance(s, torch.cuda.Stream) for s in ss)
    assert ops.streams_share_queue(ss[0], ss[0]) is True
    assert ops.streams_share_queue(ss[0], ss[1]) in (True, False)
    x = torch.ones(16, device=dev)
    with torch.cuda.stream(ss[2]):
        y = x * 2
    torch.cuda.synchronize()
    assert float(y.sum()) == 32.0


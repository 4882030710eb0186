"""hb_set_stream over a HIP runtime on host memory that writes down each call's
stream: everything after the change goes to the caller's, the change waits for
what was queued, and a graph is captured on the context's own stream."""
import ctypes
import os
import subprocess
import sys

import pytest

import host_gpu


@pytest.fixture(scope="module")
def hb(tmp_path_factory):
    """The fake runtime with its stream calls logged: (call, stream) pairs."""
    with open(os.path.join(host_gpu.ROOT, "tests", "host", "fake_hip.cpp")) as f:
        text = f.read()
    for call, at in (("hipMemcpyAsync(", "size_t n, hipMemcpyKind kind, hipStream_t) {"), ("hipStreamSynchronize(", "hipStream_t) {"),
                     ("hipEventRecord(", "hipEvent_t e, hipStream_t) {"), ("hipStreamBeginCapture(", "hipStream_t, hipStreamCaptureMode) {"),
                     ("hipGraphLaunch(", "hipGraphExec_t, hipStream_t) {"), ("hipModuleLaunchKernel(", "hipStream_t, void** args, void**) {")):
        head = text.index(at, text.index("hipError_t " + call))
        body = head + len(at)
        text = (text[:head] + at.replace("hipStream_t", "hipStream_t s_", 1) + '\n    said("%s", s_);' % call[3:-1] + text[body:])
    text = text.replace("hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {\n    *s = (hipStream_t)1;",
                        "hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {\n    *s = (hipStream_t)7;")
    text = text.replace("std::map<void*, size_t> blocks;", 'std::string log_;\nvoid said(const char* what, hipStream_t s) { log_ += std::string(what) + " " + '
                        'std::to_string((uintptr_t)s) + "\\n"; }\nstd::map<void*, size_t> blocks;')
    text = text.replace("void fake_forget(void) {", "const char* fake_log(void) { return log_.c_str(); }\nvoid fake_forget(void) {\n    log_.clear();")
    root = tmp_path_factory.mktemp("fake")
    os.makedirs(root / "tests" / "host")
    (root / "tests" / "host" / "fake_hip.cpp").write_text(text)
    mp = pytest.MonkeyPatch()
    mp.setenv("HB_CACHE_DIR", "")
    mp.setattr(host_gpu, "ROOT", str(root))
    yield host_gpu.load(tmp_path_factory.mktemp("host"))
    mp.undo()


def calls(hb):
    hb.lib.fake_log.restype = ctypes.c_char_p
    said = [line.split() for line in hb.lib.fake_log().decode().splitlines()]
    hb.lib.fake_forget()
    return [(what, int(s)) for what, s in said]


OWN = 7


@pytest.mark.parametrize("stream", [0, 1234])
def test_work_goes_to_the_set_stream(hb, stream):
    with hb.Gpu(0) as g:
        k = g.pipeline(hb.matvec_q4(128, 32, hb.Out.F32, mv_m=1))
        w, x, y = g.alloc(hb.q4_bytes(128, 32)), g.alloc(256), g.alloc(128)
        op = [hb.r(w), hb.r(x), hb.r(y)]
        calls(hb)
        g.launch(k, op, 1)
        assert calls(hb) == [("ModuleLaunchKernel", OWN)]
        g.set_stream(stream)
        assert calls(hb) == [("EventRecord", stream), ("StreamSynchronize", OWN)]
        g.set_stream(stream)
        assert calls(hb) == []
        g.launch(k, op, 1)
        g.zero(y)
        g.copy(hb.r(x, 0, 16), hb.r(y, 0, 16))
        g.download(y, "u1", 4)
        g.sync()
        g.time_ops([hb.Op(k, op, 1)], 2)
        g.time_each([hb.Op(k, op, 1)], 1)
        seen = calls(hb)
        assert {s for _, s in seen} == {stream}
        assert sum(what == "ModuleLaunchKernel" for what, _ in seen) == 5
        graph = g.graph([hb.Op(k, op, 1)])
        assert calls(hb) == [("StreamBeginCapture", OWN), ("ModuleLaunchKernel", OWN)]
        graph.launch(2)
        graph.time(1)
        seen = calls(hb)
        assert {s for _, s in seen} == {stream} and sum(what == "GraphLaunch" for what, _ in seen) == 3
        graph.free()
        calls(hb)
        g.set_stream()
        g.launch(k, op, 1)
        assert calls(hb) == [("EventRecord", OWN), ("StreamSynchronize", stream), ("ModuleLaunchKernel", OWN)]


def test_two_hip_runtimes_are_refused():
    """With torch imported last the process holds two; its null stream would be
    another than the library's."""
    code = """
import sys
sys.path.insert(0, %r)
for name in sys.argv[1:]:
    __import__(name)
import herbert_hip as hb
many = len(hb._hip_runtimes())
assert many == (1 if sys.argv[1] == "torch" else 2), hb._hip_runtimes()
g = object.__new__(hb.Gpu)
g.h = g._stream = None
hb.lib = type("lib", (), {"hb_set_stream": staticmethod(lambda h, s: 0), "hb_own_stream": staticmethod(lambda h: 0)})
g.set_stream()
try:
    g.set_stream(0)
    assert many == 1
except hb.HerbertError as e:
    assert many == 2 and "import torch before" in str(e), e
""" % os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "herbert-metal-bf16_amd")
    for order in (["torch", "herbert_hip"], ["herbert_hip", "torch"]):
        r = subprocess.run([sys.executable, "-c", code, *order], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr

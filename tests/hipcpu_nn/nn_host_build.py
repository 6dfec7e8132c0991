"""TEST INFRASTRUCTURE -- the kernel sources of csrc/nn compiled for the HOST (clang, on tests/hipcpu's stand-in for the HIP
runtime) and bound through the package's own binding, so that indexing, tiling, barriers and argument marshalling are checked
where there is no GPU.  Never imported by the package."""
import ctypes
import fcntl
import os
import re
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
CSRC = os.path.join(ROOT, "transferattack_amd", "csrc", "nn")
STAND_IN = os.path.join(ROOT, "tests", "hipcpu")
OUT = os.path.join(STAND_IN, "_build", "nn")
CLANG = "/opt/rocm/llvm/bin/clang++"


def _host_text(text):
    text = text.replace('#include "../../../include/ta_nn.h"', '#include "%s"' % os.path.join(ROOT, "include", "ta_nn.h"))
    return re.sub(r"extern __shared__ __attribute__\(\(aligned\(16\)\)\) char (\w+)\[\];", r"char* \1 = ta_nn_host::lds();", text)


def build():
    os.makedirs(OUT, exist_ok=True)
    lib = os.path.join(OUT, "libta_nn_host.so")
    sources = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
    headers = sorted(f for f in os.listdir(CSRC) if f.endswith(".h") and f != "ta_nn_mma.h")
    deps = [os.path.join(CSRC, f) for f in sources + headers] + [os.path.join(HERE, f) for f in ("ta_nn_mma.h", "nn_host_build.py")]
    deps += [os.path.join(ROOT, "include", "ta_nn.h"), os.path.join(STAND_IN, "hipcpu.cpp")]
    fresh = lambda: os.path.exists(lib) and all(os.path.getmtime(d) <= os.path.getmtime(lib) for d in deps)   # noqa: E731
    if fresh():
        return lib
    with open(os.path.join(OUT, ".lock"), "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        if fresh():
            return lib
        for h in headers:
            with open(os.path.join(OUT, h), "w") as fh:
                fh.write(_host_text(open(os.path.join(CSRC, h)).read()))
        flags = ["-O1", "-std=c++17", "-fPIC", "-w", "-pthread", "-D__builtin_elementwise_fma=hipcpu_elementwise_fma", "-I", HERE, "-I", OUT,
                 "-I", STAND_IN]
        jobs = []
        for src in sources:
            cpp = os.path.join(OUT, src.replace(".hip", ".cpp"))
            with open(cpp, "w") as fh:
                fh.write(_host_text(open(os.path.join(CSRC, src)).read()))
                if src == "runtime.hip":
                    fh.write('\nnamespace ta_nn_host { char* lds() { alignas(64) static thread_local char a[163840]; return a; } }\n')
            jobs.append((cpp, cpp.replace(".cpp", ".o")))
        jobs.append((os.path.join(STAND_IN, "hipcpu.cpp"), os.path.join(OUT, "hipcpu.o")))
        running = [subprocess.Popen([CLANG] + flags + ["-c", c, "-o", o], stderr=subprocess.PIPE, text=True) for c, o in jobs]
        for p, (c, _) in zip(running, jobs):
            err = p.communicate()[1]
            assert p.returncode == 0, (c, err[-3000:])
        tmp = "%s.%d.tmp" % (lib, os.getpid())
        subprocess.run([CLANG, "-shared", "-pthread", "-o", tmp] + [o for _, o in jobs], check=True, capture_output=True, text=True)
        os.replace(tmp, lib)
    return lib


_lib = None


def install(monkeypatch):
    """the package's binding on the host build, CPU tensors allowed, for one test"""
    global _lib
    from transferattack_amd import _nn
    if _lib is None:
        _lib = _nn.bind(ctypes.CDLL(build()))
    monkeypatch.setattr(_nn, "_lib", _lib)
    monkeypatch.setattr(_nn, "_on_device", lambda t, name: None)
    monkeypatch.setattr(_nn, "_launch", lambda name, like, *args: _nn._check(getattr(_lib, name)(*args, None), name))

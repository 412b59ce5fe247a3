"""In-tree build of libdsuf_qmm.so (nvcc, sm_100a only) and, where torch can be imported, of the Python module dsuf_hostcall.so (g++).

``python deepseek-ultrafast_b200/build.py`` or ``build()`` from Python.  Objects are cached under
``csrc/build/`` and rebuilt when a source or header is newer.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libdsuf_qmm.so")
HOSTCALL = os.path.join(HERE, "dsuf_hostcall.so")
HOSTCALL_FOR = os.path.join(CSRC, "build", "hostcall.for")     # the torch and Python that the module was built for
SOURCES = ["abi.cu", "quant.cu", "moe_aux.cu", "stream_launch.cu", "noalloc.cu", "ep_comm.cu", "peak_probe.cu", "lm_head.cu", "kv_cache.cu", "attn_decode.cu", "attn_prompt.cu", "sample.cu", "pack.cc", "loader.cc"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
         "-Xptxas", "-v", "--expt-relaxed-constexpr", "-ccbin", "/usr/bin/g++"] + os.environ.get("DSUF_EXTRA_NVCC_FLAGS", "").split()


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs.append(os.path.join(HERE, "..", "include", "dsuf_qmm.h"))
    return hs


def _compile(src, obj, log):
    cmd = [NVCC, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    if src.endswith(".cc"):
        cmd = [NVCC, "-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-ccbin", "/usr/bin/g++", "-x", "cu", "-c",
               os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    with open(log, "w") as f:
        f.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")


def build_hostcall():
    """dsuf_hostcall.so: the Python entries that check tensors and call the library in native code (csrc/hostcall.cc), against the torch and Python
    that run this.  None without torch, or with one that has no CUDA: the library itself needs neither."""
    import importlib.util
    import sysconfig
    if importlib.util.find_spec("torch") is None:
        return None
    import torch
    if torch.version.cuda is None:
        return None
    src, header = os.path.join(CSRC, "hostcall.cc"), os.path.join(HERE, "..", "include", "dsuf_qmm.h")
    made_for = f"torch {torch.__version__} in {os.path.dirname(torch.__file__)}, Python {sys.version}\n"
    if os.path.exists(HOSTCALL) and os.path.getmtime(HOSTCALL) >= max(os.path.getmtime(src), os.path.getmtime(header)):
        try:
            with open(HOSTCALL_FOR) as f:
                if f.read() == made_for:
                    return HOSTCALL
        except OSError:
            pass
    root = os.path.dirname(torch.__file__)
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include")]
    cuda = os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", cuda,
           "-I", sysconfig.get_paths()["include"], *[x for d in includes for x in ("-isystem", d)], src, "-o", HOSTCALL + ".tmp",
           "-L", os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed on hostcall.cc:\n" + r.stderr)
    os.replace(HOSTCALL + ".tmp", HOSTCALL)
    os.makedirs(os.path.dirname(HOSTCALL_FOR), exist_ok=True)
    with open(HOSTCALL_FOR, "w") as f:
        f.write(made_for)
    return HOSTCALL


def build(verbose=False):
    bdir = os.path.join(CSRC, "build")
    os.makedirs(bdir, exist_ok=True)
    newest_h = max(os.path.getmtime(h) for h in _headers())
    jobs, objs = [], []
    for s in SOURCES:
        if not os.path.exists(os.path.join(CSRC, s)):
            continue
        obj = os.path.join(bdir, s + ".o")
        objs.append(obj)
        src_m = max(os.path.getmtime(os.path.join(CSRC, s)), newest_h)
        if not os.path.exists(obj) or os.path.getmtime(obj) < src_m:
            jobs.append((s, obj, os.path.join(bdir, s + ".log")))
    if jobs:
        with ThreadPoolExecutor(max_workers=8) as ex:
            list(ex.map(lambda j: _compile(*j), jobs))
    if jobs or not os.path.exists(OUT):
        # link beside the target and rename: a reader never sees a half-written library
        cmd = [NVCC, "-shared", "-o", OUT + ".tmp", *objs, "-ccbin", "/usr/bin/g++", "-lcudart", "-lpthread"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("link failed:\n" + r.stdout + r.stderr)
        os.replace(OUT + ".tmp", OUT)
    build_hostcall()
    if verbose:
        for s, _, log in jobs:
            print(open(log).read())
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))

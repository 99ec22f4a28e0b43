"""The serving-step operators' host code over a stand-in for the CUDA runtime (fake_device.cpp): which launches a call
makes, with which cut, and what happens when one fails.  No GPU; the kernels are compiled to PTX only and never run."""
import ctypes as C
import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "compressed-kv-attention_b200", "csrc")
OUT = os.path.join(HERE, "_build")
SOURCES = [os.path.join(CSRC, f) for f in ("attention.cu", "codec.cu", "batch.cu", "rotate.cu", "paged_stream.cu",
                                              "prefix_attention.cu")] + [
    os.path.join(HERE, "fake_device.cu"), os.path.join(HERE, "fake_device.cpp")]
KINDS = ["rotate", "prefix", "stream", "combine", "other"]


class Launch(C.Structure):
    _fields_ = [(n, C.c_int32) for n in (
        "kind_index", "device", "grid", "threads", "smem", "allowed", "counter", "prefix_tiles", "n_split", "split_tiles",
        "row_groups", "stream_ctas", "stream_runs", "shared_runs", "rows")]

    @property
    def kind(self):
        return KINDS[self.kind_index]


def nvcc():
    path = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    return path if os.path.exists(path) else shutil.which("nvcc")


def build():
    os.makedirs(OUT, exist_ok=True)
    lib = os.path.join(OUT, "libbatch_host.so")
    deps = SOURCES + [os.path.join(HERE, "fake_device.h")] + [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [
        os.path.join(CSRC, "..", "..", "include", "kvexp_b200.h"), os.path.abspath(__file__)]
    if os.path.exists(lib) and all(os.path.getmtime(f) <= os.path.getmtime(lib) for f in deps):
        return lib
    tag = str(os.getpid())
    objs = [os.path.join(OUT, os.path.basename(s) + "." + tag + ".o") for s in SOURCES]
    flags = ["-std=c++17", "-gencode", "arch=compute_100a,code=compute_100a", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
             "-ccbin", "/usr/bin/g++"]
    jobs = [subprocess.Popen([nvcc(), *flags, "-c", s, "-o", o]) for s, o in zip(SOURCES, objs)]
    assert [j.wait() for j in jobs] == [0] * len(jobs)
    # the library's own symbols first: a CUDA runtime may be loaded in this process
    subprocess.run(["/usr/bin/g++", "-shared", "-Wl,-Bsymbolic", "-Wl,--no-undefined", "-o", lib + tag, *objs], check=True)
    os.replace(lib + tag, lib)
    for o in objs:
        os.remove(o)
    return lib


def load(kvx):
    """The library, with the signatures of the entry points and of the stand-in's controls."""
    lib = C.CDLL(build())
    lib.kvx_batch_create.argtypes = [C.c_int] * 5 + [C.POINTER(C.c_void_p)]
    lib.kvx_batch_destroy.argtypes = [C.c_void_p]
    lib.kvx_batch_destroy.restype = None
    lib.kvx_batch_attend.argtypes = [C.c_void_p, C.POINTER(kvx.kvx_attend), C.c_void_p]
    lib.kvx_batch_append.argtypes = [C.c_void_p] + [C.POINTER(kvx.kvx_view)] * 4 + [
        C.c_int, C.POINTER(kvx.kvx_rope), C.c_void_p, C.POINTER(kvx.kvx_pages), C.c_void_p]
    lib.kvx_batch_rotate.argtypes = [C.c_void_p] + [C.POINTER(kvx.kvx_view)] * 2 + [
        C.c_int, C.c_int, C.POINTER(kvx.kvx_rope), C.c_int, C.c_void_p]
    lib.kvx_batch_wait_limit.argtypes = [C.c_void_p, C.c_int]
    lib.kvx_batch_check.argtypes = [C.c_void_p]
    lib.fake_last_error.restype = C.c_char_p
    lib.fake_set_error.argtypes = [C.c_char_p]
    lib.fake_prefix.restype = C.c_void_p
    lib.fake_prefix_free.argtypes = [C.c_void_p]
    lib.fake_launches.argtypes = [C.POINTER(Launch), C.c_int]
    return lib


class Device:
    """A fresh stand-in and calls with made-up addresses."""

    def __init__(self, kvx):
        self.kvx, self.lib = kvx, load(kvx)
        self.lib.fake_reset()

    def create(self, max_batch, hq, hkv, dim, dtype=0):
        h = C.c_void_p()
        rc = self.lib.kvx_batch_create(max_batch, hq, hkv, dim, dtype, C.byref(h))
        return rc, h

    def attend(self, h, batch, hq, hkv, dim, prefix_len=0, max_len=0, page_tokens=16, coded=None):
        k = self.kvx
        at = 1 << 20
        pages = k.kvx_pages(at, at, page_tokens * hkv * dim, hkv * dim, dim, 1 << 20, page_tokens)
        x = k.kvx_attend(q=k.kvx_view(at, hq * dim, dim), out=k.kvx_view(at, hq * dim, dim), lse=None,
                         pages=C.addressof(pages), prefix_table=at if prefix_len else None, prefix=coded,
                         table=at, lens=at, table_stride=1 << 20, prefix_len=prefix_len, max_len=max_len, batch=batch, scale=0.0)
        return self.lib.kvx_batch_attend(h, C.byref(x), None)

    def rotate(self, h, tokens, heads, dim):
        k = self.kvx
        at = 1 << 20
        v, r = k.kvx_view(at, heads * dim, dim), k.kvx_rope(at, at, at, None, 0, 100, dim, 1, 0)
        return self.lib.kvx_batch_rotate(h, C.byref(v), C.byref(v), tokens, heads, C.byref(r), 0, None)

    def append(self, h, tokens, hkv, dim):
        k = self.kvx
        at = 1 << 20
        v, p = k.kvx_view(at, hkv * dim, dim), k.kvx_pages(at, at, 16 * hkv * dim, hkv * dim, dim, 100, 16)
        return self.lib.kvx_batch_append(h, None, C.byref(v), C.byref(v), None, tokens, None, at, C.byref(p), None)

    def launches(self):
        buf = (Launch * 4096)()
        return list(buf[:self.lib.fake_launches(buf, 4096)])

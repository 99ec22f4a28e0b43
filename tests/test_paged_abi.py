"""CPU checks of the serving-step entry points: argument errors come before any CUDA call."""
import ctypes as C

import pytest


@pytest.mark.parametrize("args", [(0, 4, 2, 64, 0), (70000, 4, 2, 64, 0), (1, 4, 3, 64, 0), (1, 0, 1, 64, 0),
                                  (1, 4, 0, 64, 0), (1, 4, 2, 63, 0), (1, 4, 2, 258, 0), (1, 4, 2, 0, 0), (1, 4, 2, 64, 2)])
def test_batch_create_refuses(kvx, args):
    h = C.c_void_p()
    assert kvx._batch_create(*args, C.byref(h)) == kvx.KVX_ERR_INVALID_ARGUMENT
    assert b"kvx_batch_create" in kvx._last_error() and not h.value


def test_null_handles(kvx):
    v = bytes(kvx.kvx_view(16, 64, 64))
    r = bytes(kvx.kvx_rope(16, 16, 16, None, 0, 1, 64, 1, 0))
    p = bytes(kvx.kvx_pages(16, 16, 64, 64, 64, 1, 1))
    assert kvx._batch_rotate(None, v, v, 1, 1, r, 0, None) == kvx.KVX_ERR_INVALID_ARGUMENT
    assert kvx._batch_append(None, None, v, v, None, 1, None, 16, p, None) == kvx.KVX_ERR_INVALID_ARGUMENT
    assert kvx._batch_attend(None, bytes(kvx.kvx_attend()), None) == kvx.KVX_ERR_INVALID_ARGUMENT
    assert kvx._batch_check(None) == kvx.KVX_ERR_INVALID_ARGUMENT
    kvx._batch_destroy(None)


def test_host_tensors_are_refused(kvx):
    import torch
    x = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        kvx.Pages(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        kvx.Rope(torch.zeros((4, 32)), torch.zeros((4, 32)))
    with pytest.raises(ValueError, match="dtype"):
        kvx.Batch(1, 1, 1, 64, dtype="fp32")


@pytest.mark.parametrize("args", [(2049, 8, 2, 64, 0), (1, 65538, 2, 64, 0)])
def test_batch_create_refuses_what_it_cannot_count(kvx, args):
    """More sequences or heads than the streaming kernel's lists and the grids are for."""
    h = C.c_void_p()
    assert kvx._batch_create(*args, C.byref(h)) == kvx.KVX_ERR_INVALID_ARGUMENT and not h.value


def test_wait_limit_of_no_batch(kvx):
    assert kvx._batch_wait_limit(None, 1) == kvx.KVX_ERR_INVALID_ARGUMENT


class _OnDevice:
    """What the binding looks at of a CUDA tensor."""

    def __init__(self, device, dtype, *shape):
        import torch
        self.device, self.dtype, self.shape, self.is_cuda = device, dtype, torch.Size(shape), True

    def get_device(self):
        return self.device

    def stride(self, i=None):
        st = [1]
        for n in self.shape[:0:-1]:
            st.insert(0, st[0] * n)
        return tuple(st) if i is None else st[i]

    def data_ptr(self):
        return 1 << 20

    def is_contiguous(self):
        return True


def test_tensors_of_another_device_are_refused(kvx):
    """Nothing reaches the library from a tensor, tables or pools that are not on the batch's device."""
    import torch
    bf, f32, i32, i64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
    T = _OnDevice
    with pytest.raises(ValueError, match="sin is on device 1"):
        kvx.Rope(T(0, f32, 9, 32), T(1, f32, 9, 32))
    with pytest.raises(ValueError, match="axis is on device 0"):
        kvx.Rope(T(1, f32, 9, 32), T(1, f32, 9, 32), axis=T(0, torch.uint8, 32), n_axes=2)
    with pytest.raises(ValueError, match="v is on device 1"):
        kvx.Pages(T(0, bf, 9, 16, 2, 64), T(1, bf, 9, 16, 2, 64))
    b = object.__new__(kvx.Batch)  # (no device here to make one on)
    b._h, b.device, b.n_q_heads, b.n_kv_heads, b.dim = None, 0, 4, 2, 64
    b._type, b._int32, b._int64, b._float32 = bf, i32, i64, f32
    rope, pages = kvx.Rope(T(0, f32, 9, 32), T(0, f32, 9, 32)), kvx.Pages(T(0, bf, 9, 16, 2, 64), T(0, bf, 9, 16, 2, 64))
    x, kv = T(0, bf, 3, 4, 64), T(0, bf, 3, 2, 64)

    def rotate(**k):
        a = dict(x=x, pos=T(0, i32, 3), rope=rope, out=x) | k
        b.rotate(a["x"], a["pos"], a["rope"], a["out"])

    def append(**k):
        a = dict(q=x, k=kv, v=kv, pos=T(0, i32, 3), rope=rope, slots=T(0, i64, 3), pages=pages, q_out=x) | k
        b.append(**a)

    def attend(**k):
        a = dict(q=x, out=x, pages=pages, table=T(0, i32, 3, 1), lens=T(0, i32, 3), max_len=16, prefix_table=T(0, i32, 2),
                 prefix_len=20, lse=T(0, f32, 3, 4)) | k
        b.attend(a.pop("q"), a.pop("out"), a.pop("pages"), a.pop("table"), a.pop("lens"), a.pop("max_len"), **a)

    far_rope = kvx.Rope(T(1, f32, 9, 32), T(1, f32, 9, 32))
    far_pages = kvx.Pages(T(1, bf, 9, 16, 2, 64), T(1, bf, 9, 16, 2, 64))
    far = {"x": T(1, bf, 3, 4, 64), "kv": T(1, bf, 3, 2, 64), "pos": T(1, i32, 3)}
    for call, bad in [(rotate, [("x", far["x"]), ("out", far["x"]), ("pos", far["pos"]), ("rope", far_rope)]),
                      (append, [("q", far["x"]), ("k", far["kv"]), ("v", far["kv"]), ("q_out", far["x"]), ("pos", far["pos"]),
                                ("slots", T(1, i64, 3)), ("rope", far_rope), ("pages", far_pages)]),
                      (attend, [("q", far["x"]), ("out", far["x"]), ("pages", far_pages), ("table", T(1, i32, 3, 1)),
                                ("lens", far["pos"]), ("prefix_table", T(1, i32, 2)), ("lse", T(1, f32, 3, 4))])]:
        with pytest.raises(ValueError, match="bad argument"):  # what the library says of no handle: every tensor was taken
            call()
        for name, value in bad:
            with pytest.raises(ValueError, match="on device 1, not on device 0"):
                call(**{name: value})

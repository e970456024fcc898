"""The 8-bit cache's entries refuse tensors that are not on the handle's device, each of
them, before anything is launched."""
import ctypes as C

import pytest
import torch

from ttsxabe_b200 import Gpu, InvalidArgument


class Tensor:
    """What the entries look at of a tensor."""

    def __init__(self, dtype=torch.float32, device=0, contiguous=True, n=1 << 16):
        self.dtype, self.device, self.contiguous, self.n = dtype, device, contiguous, n

    def get_device(self):
        return self.device

    def is_contiguous(self):
        return self.contiguous

    def numel(self):
        return self.n

    def element_size(self):
        return torch.empty(0, dtype=self.dtype).element_size()

    def stride(self):
        return (1,) if self.contiguous else (2,)

    def data_ptr(self):
        return 1 << 20


class Library:
    """Stands in for the shared library: counts what reaches it."""

    def __init__(self):
        self.calls = 0

    def __getattr__(self, name):
        def call(*args):
            self.calls += 1
            return 0
        return call


class Scratch:
    def _bind(self, gpu):
        return None


def handle():
    g = Gpu.__new__(Gpu)
    g._h, g.ordinal, g._lib = None, 0, Library()
    g.uninit = lambda n: Tensor()
    return g


def i32s(*xs):
    return (C.c_int32 * len(xs))(*xs)


TABLE = (C.c_void_p * 1)(1 << 20)
F16, I32, U8 = torch.float16, torch.int32, torch.uint8
CALLS = {
    "append": (lambda g, q, k, v, f, o: g.rope_append_q8(q, k, v, i32s(0, 1), TABLE, i32s(64), i32s(0), i32s(0), f, 4, 2, 64, q_out=o),
               [torch.float32] * 5),
    "decode": (lambda g, q, o: g.decode_batched_q8(q, TABLE, i32s(1), i32s(64), 4, 2, 64, 0.1, Scratch(), out=o), [torch.float32, F16]),
    "flash": (lambda g, q, o: g.flash_attn_q8(q, i32s(0, 1), TABLE, i32s(64), i32s(0), 4, 2, 64, 0.1, True, out=o), [torch.float32, F16]),
    "read": (lambda g, k, v: g.cache_read_q8(TABLE, i32s(64), i32s(1), i32s(0), i32s(0, 1), 2, 64, k_out=k, v_out=v), [F16, F16]),
    "evict": (lambda g, i: g.cache_evict_q8(TABLE, i32s(64), TABLE, i32s(64), i32s(40), i32s(0), 0, 0, 2, 64, index=i), [I32]),
    "grow": (lambda g, s, d: g.cache_grow_q8(s, d, 2, 64, 64, 128, 1), [U8, U8]),
    "inv_freq": (lambda g, d: g.rope_inv_freq(1e4, 64, d), [torch.float32]),
}


@pytest.mark.parametrize("name", CALLS)
def test_every_tensor_is_looked_at(name):
    call, types = CALLS[name]
    g = handle()
    call(g, *(Tensor(t) for t in types))
    assert g._lib.calls == 1
    for i in range(len(types)):
        for device in (1, -1):
            args = [Tensor(t) for t in types]
            args[i].device = device
            with pytest.raises(InvalidArgument, match="not cuda:0"):
                call(g, *args)
        args = [Tensor(t) for t in types]
        args[i].contiguous = False
        with pytest.raises(InvalidArgument):
            call(g, *args)
    assert g._lib.calls == 1


def test_host_tensors_are_refused():
    g = handle()
    q, k = torch.zeros(256), torch.zeros(128)
    with pytest.raises(InvalidArgument, match="a tensor on cpu"):
        g.rope_append_q8(q, k, k, i32s(0, 1), TABLE, i32s(64), i32s(0), i32s(0), None, 4, 2, 64)
    with pytest.raises(InvalidArgument, match="a tensor on cpu"):
        g.decode_batched_q8(q, TABLE, i32s(1), i32s(64), 4, 2, 64, 0.1, Scratch())
    assert g._lib.calls == 0


def test_divisors_of_the_frequencies():
    for d in (Tensor(torch.float64), Tensor(n=31), Tensor(contiguous=False)):
        with pytest.raises(InvalidArgument, match="divisors"):
            handle().rope_inv_freq(1e4, 64, d)

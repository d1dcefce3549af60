"""The memory-over-ticks operators' errors on the host. Without a GPU."""
import contextlib
import ctypes
import subprocess

import pytest

from flyguy_b200 import memory, native


def test_a_refused_size_is_refused_in_the_same_words_again():
    """A workspace's size is kept from call to call; a refusal's words are the refusal's each time, also after a call that went
    well."""
    good, bad = (1, 8, 2, 2, 64, 64, 0), (1, 8, 2, 2, 300, 64, 0)
    for _ in range(3):
        with pytest.raises(native.FlyguyError, match="dim and value_dim must be 1 to 256"):
            memory._room(memory._decay_room(bad, False, False), None)
        assert native.lib().fg_decay_work(memory._DECAY.pack(*(0,) * 38, *good, 1.0, 0, 0), 0) == 0
        assert native.lib().fg_mem_last_error() == b""


def test_kernels_are_set_up_on_every_device(tmp_path):
    """fg_once.h: once a device, on each device, again after a failure; numbers past 63 each time."""
    src = tmp_path / "once.cpp"
    src.write_text("""
#include "fg_once.h"
extern "C" int setups(const int* devices, const int* fails, int n, int* ran) {
    fgm::OnEachDevice here;
    int thrown = 0;
    for (int i = 0; i < n; ++i) {
        ran[i] = 0;
        try {
            here.first(devices[i], [&] { ran[i] = 1; if (fails[i]) throw 1; });
        } catch (int) { ++thrown; }
    }
    return thrown;
}
""")
    lib = tmp_path / "once.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(native.PKG / "csrc"), "-o", str(lib), str(src)], check=True)
    devices, fails = [0, 0, 1, 1, 0, 63, 63, 64, 64, 2, 2, 2], [0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 0, 0]
    n = len(devices)
    ran = (ctypes.c_int * n)()
    assert ctypes.CDLL(str(lib)).setups((ctypes.c_int * n)(*devices), (ctypes.c_int * n)(*fails), n, ran) == 1
    assert list(ran) == [1, 0, 1, 0, 0, 1, 0, 1, 1, 1, 1, 0]


def test_no_kernel_is_set_up_once_for_all_devices():
    """Attributes are set at every launch or by OnEachDevice, never behind a flag of the process."""
    for f in ("fg_decay.cu", "fg_decay_mma.cuh", "fg_decay_tc.cuh", "fg_rotate.cu"):
        text = (native.PKG / "csrc" / f).read_text()
        assert "static const bool" not in text and "static bool" not in text, f


def test_a_wait_that_ran_out_is_told(monkeypatch):
    """memory.sync on a library whose fg_mem_sync reports a wait that ran out, and on one that reports none."""
    class Library:
        status, asked = 0, []

        def fg_mem_sync(self, stream):
            self.asked.append(stream)
            return self.status

        def fg_mem_last_error(self):
            return b"fg_decay_attn: a wait on the tensor cores ran out"

    fake = Library()
    monkeypatch.setattr(memory, "lib", lambda: fake)
    monkeypatch.setattr(memory, "_raw_stream", lambda device: 7)
    monkeypatch.setattr(memory, "_device", lambda: 0)
    monkeypatch.setattr(memory.torch.cuda, "device", lambda device: contextlib.nullcontext())
    memory.sync()
    fake.status = -1
    with pytest.raises(native.FlyguyError, match="ran out"):
        memory.sync()
    assert fake.asked == [7, 7]

"""The memory-over-ticks operators without a GPU: the rotation's plan, and argument errors as statuses."""
import ctypes
import math

import pytest
import torch

from flyguy_b200 import memory, native


@pytest.mark.parametrize("turned", [2, 64, 128])
def test_turns_are_the_frequencies(turned):
    """Against Python's doubles: the power's exponent is rounded at 2^-53 times ln(10000) = 9.2, and the quotient is; one
    unit of 2^-64 of a turn for the rounding to integers."""
    t = memory.rotary_turns(turned)
    for i, x in enumerate(t.tolist()):
        f = 10000.0 ** (-2 * i / turned) / (2 * math.pi) * 2.0 ** 64
        assert abs(x - f) <= 16 * 2.0 ** -53 * f + 1
    assert memory.rotary_turns(0).numel() == 0


def test_turns_for_longer_recordings():
    """Whole numbers of 2^-64 of a turn: each is half a unit off at most, a quotient of two by one in all (and by the
    doubles they are compared in, 2^-52 of the value)."""
    plain = memory.rotary_turns(64).double()
    near = lambda a, b: bool(((a - b).abs() <= 1 + b * 2.0 ** -52).all())   # noqa: E731
    assert near(memory.rotary_turns(64, scaling="linear", factor=8).double(), plain / 8)
    base = memory.rotary_turns(64, scaling="base", factor=8).double()
    assert base[0] == plain[0] and near(base[-1:], plain[-1:] / 8) and (base[1:] < plain[1:]).all()
    parts = memory.rotary_turns(64, scaling="parts", factor=8, original=1024).double()
    turns = plain / 2.0 ** 64 * 1024
    assert torch.equal(parts[turns > 32], plain[turns > 32])
    assert near(parts[turns < 1], plain[turns < 1] / 8)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((parts < plain) & (parts > plain / 8))[between].all()


def test_argument_structures_match_the_header():
    """The packed fields are the header's: 8 bytes each, one per declared name."""
    import re
    text = (native.PKG.parent / "include" / "flyguy_b200.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, packed in (("fg_rotate_args", memory._ROTATE), ("fg_decay_args", memory._DECAY), ("fg_step_args", memory._STEP)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        n = 0
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            each = 4 if decl.startswith("fg_ticks") else 1
            for field in decl.split(","):
                n += each * (2 if "[2]" in field else 1)
        assert packed.size == 8 * n, name


def test_argument_errors_are_statuses():
    L = native.lib()
    assert L.fg_norm_rotate(None, None) == -1 and "no arguments" in L.fg_mem_last_error().decode()
    assert L.fg_decay_attn(None, None) == -1 and L.fg_decay_attn_bwd(None, None) == -1 and L.fg_decay_step(None, None) == -1
    assert L.fg_decay_work(None, 0) == -1
    zero = bytes(memory._DECAY.size)
    assert L.fg_decay_attn(zero, None) == -1 and "heads" in L.fg_mem_last_error().decode()
    fields = [0] * 32 + [0] * 6 + [2, 3, 4, 2, 64, 64, 0] + [1.0, 0, 0]
    assert L.fg_decay_attn(memory._DECAY.pack(*fields), None) == -1
    assert "log_decay" in L.fg_mem_last_error().decode()
    assert L.fg_decay_work(memory._DECAY.pack(*fields), 1) > 0               # shared heads' gradients need room
    rot = [0] * 32 + [0] * 6 + [1, 0] + [2, 3, 64, 63, 0, 0, 0, 0, 8, 0, 0, 0] + [1.0, 1.0, 0, 0]
    assert L.fg_norm_rotate(memory._ROTATE.pack(*rot), None) == -1 and "even" in L.fg_mem_last_error().decode()
    rot[43] = 64
    assert L.fg_norm_rotate(memory._ROTATE.pack(*rot), None) == -1 and "turns" in L.fg_mem_last_error().decode()


def test_outputs_that_inputs_still_need_are_refused():
    """gstate is written while another of the gradients' scans still reads the states; an eps that is 0 in fp32 is none."""
    L = native.lib()
    for other in (33, 35):                                                   # state, gstate_out
        fields = [0] * 32 + [0] * 6 + [0, 0, 4, 4, 64, 64, 0] + [1.0, 0, 0]
        fields[32], fields[36], fields[other] = 16, 256, 256
        assert L.fg_decay_attn_bwd(memory._DECAY.pack(*fields), None) == -1
        assert "gstate" in L.fg_mem_last_error().decode()
    rot = [0] * 32 + [0] * 6 + [1, 0] + [0, 0, 64, 0, 0, 0, 0, 0, 8, 0, 0, 1] + [1e-60, 1.0, 0, 0]
    assert L.fg_norm_rotate(memory._ROTATE.pack(*rot), None) == -1 and "eps" in L.fg_mem_last_error().decode()


def test_the_workspace_holds_its_parts():
    """Heads' states of 9 floats in parts, then the shared heads' results: each begins at 16 bytes and all of it fits."""
    L = native.lib()
    sizes = [1, 4096, 2, 1, 3, 3, 0]                                         # few long recordings are split
    pack = lambda heads, keys: memory._DECAY.pack(*[0] * 38, *sizes[:2], heads, keys, *sizes[4:], 1.0, 0, 0)  # noqa: E731
    for heads in (1, 2, 3, 5):
        states = L.fg_decay_work(pack(heads, heads), 1)
        assert states > 0 and states % 16 == 0
        one = -(-4096 * heads * 3 * 4 // 16) * 16
        assert L.fg_decay_work(pack(heads, 1), 1) == states + (2 * one if heads > 1 else 0)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 2, 8)
    for fn, args in ((memory.rotate, (x, memory.rotary_turns(8))), (memory.norm_rotate, (x, x)),
                     (memory.decay_attention, (x, x, x, torch.zeros(2))),
                     (memory.decay_step, (x[0], x[0], x[0], torch.zeros(2), torch.zeros(2, 2, 8, 8)))):
        with pytest.raises(native.FlyguyError, match="CUDA"):
            fn(*args)

"""The delta rule, layer norm and dropout without a GPU: argument structures, errors as statuses, and the generator that the GPU
tests take for true."""
import re

import numpy as np
import pytest

from flyguy_b200 import delta, layers, native


def philox(counter, key):
    """Philox4x32-10: four words of arrays of counters, as unsigned 64-bit integers below 2^32."""
    low, half = np.uint64(0xffffffff), np.uint64(32)
    c, k = [np.asarray(x, np.uint64) for x in counter], [int(x) for x in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def test_the_generator_is_the_published_one():
    """Known answers of the generator's authors (counter and key of zeros, of ones)."""
    assert [int(x) for x in philox([0] * 4, [0] * 2)] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert [int(x) for x in philox([0xffffffff] * 4, [0xffffffff] * 2)] == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


def test_argument_structures_match_the_header():
    text = (native.PKG.parent / "include" / "flyguy_b200.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, packed in (("fg_delta_args", delta._DELTA), ("fg_delta_step_args", delta._STEP), ("fg_norm_args", layers._NORM),
                         ("fg_dropout_args", layers._DROPOUT)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        n = 0
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            n += (4 if decl.startswith("fg_ticks") else 1) * len(decl.split(","))
        assert packed.size == 8 * n, name


def _error():
    return native.lib().fg_mem_last_error().decode()


def _delta(sizes, offsets=0, work=(0, 0), **pointers):
    """fg_delta_args with these sizes (batch, ticks, heads, query / key / value heads, dim, value_dim, type), pointers by field number."""
    f = [0] * 52
    for at, p in pointers.items():
        f[int(at[1:])] = p
    return delta._DELTA.pack(*f, offsets, *sizes, 1.0, *work)


GOOD = (2, 100, 4, 4, 2, 2, 64, 64, 1)


def test_no_arguments_are_an_error():
    L = native.lib()
    for fn in (L.fg_delta_attn, L.fg_delta_attn_bwd, L.fg_delta_step, L.fg_layer_norm, L.fg_layer_norm_bwd, L.fg_dropout):
        assert fn(None, None) == -1 and "no arguments" in _error()
    assert L.fg_delta_work(None, 0) == -1 and L.fg_layer_norm_work(None) == -1


@pytest.mark.parametrize("at, value, words", [
    (0, -1, "negative"), (1, -5, "negative"), (2, 0, "multiple"), (3, 3, "multiple"), (4, 0, "multiple"), (5, 8, "multiple"), (6, 0, "dim must be"),
    (6, 129, "dim must be"), (7, 257, "value_dim 1 to 256"), (7, 0, "value_dim"), (8, 3, "unknown type"), (0, 1 << 40, "too many"), (1, 1 << 50, "too many"),
    (0, (1 << 63) - 1, "too many"), (1, (1 << 63) - 1, "too many"), (1, 1 << 36, "too many")])
def test_refused_sizes(at, value, words):
    L = native.lib()
    sizes = (*GOOD[:at], value, *GOOD[at + 1:])
    for _ in range(2):
        assert L.fg_delta_work(_delta(sizes), 1) == -1 and words in _error()
        assert L.fg_delta_attn(_delta(sizes), None) == -1 and words in _error()
        assert L.fg_delta_attn_bwd(_delta(sizes), None) == -1 and words in _error()
        assert L.fg_delta_work(_delta(GOOD), 1) > L.fg_delta_work(_delta(GOOD), 0) > 0 and _error() == ""


def test_refused_pointers_and_workspaces():
    L = native.lib()
    assert L.fg_delta_attn(_delta(GOOD), None) == -1 and "null pointer" in _error()
    some = {f"f{4 * i}": 4096 for i in range(12)}
    assert L.fg_delta_attn(_delta(GOOD, **some), None) == -1 and "workspace is too small" in _error()
    size = L.fg_delta_work(_delta(GOOD), 0)
    assert L.fg_delta_attn(_delta(GOOD, work=(4096, size - 1), **some), None) == -1 and "workspace is too small" in _error()
    assert L.fg_delta_attn(_delta(GOOD, work=(4097, size), **some), None) == -1 and "16-byte aligned" in _error()
    same = some | {"f48": 512, "f49": 512}
    assert L.fg_delta_attn(_delta(GOOD, work=(4096, size), **same), None) == -1 and "state_out are the same" in _error()
    same = some | {"f48": 512, "f51": 512}
    assert L.fg_delta_attn_bwd(_delta(GOOD, work=(4096, size), **same), None) == -1 and "gstate is state" in _error()


def test_what_is_held():
    L = native.lib()
    some = {f"f{4 * i}": 4096 for i in range(12)}
    held = L.fg_delta_held(_delta(GOOD))
    assert held > 0 and L.fg_delta_held(None) == -1 and L.fg_delta_held(_delta((-1, *GOOD[1:]))) == -1
    work = [L.fg_delta_work(_delta(GOOD), which) for which in range(4)]
    assert work[2] < work[0] and work[3] < work[1] <= work[3] + held
    for fn, size in ((L.fg_delta_attn_hold, work[2]), (L.fg_delta_attn_bwd_held, work[3])):
        args = _delta(GOOD, work=(4096, size), **some)
        assert fn(None, 4096, held, None) == -1 and "no arguments" in _error()
        assert fn(args, 4096, held - 1, None) == -1 and "held is too small" in _error()
        assert fn(args, None, held, None) == -1 and "held is too small" in _error()
        assert fn(args, 4097, held, None) == -1 and "held is not 16-byte aligned" in _error()
    assert L.fg_delta_attn_bwd_held(_delta(GOOD, work=(4096, work[3] - 1), **some), 4096, held, None) == -1 and "workspace is too small" in _error()


def test_a_workspace_is_the_recordings_slots_and_nothing_more():
    """Packed recordings take at most a slot more each than their ticks do; parts only where recordings are few and long."""
    L = native.lib()
    whole, packed = L.fg_delta_work(_delta(GOOD), 0), L.fg_delta_work(_delta((2, 200, *GOOD[2:]), offsets=8), 0)
    assert whole <= packed <= 2 * whole
    long, split = (64, 65536, *GOOD[2:]), (1, 65536, *GOOD[2:])
    assert L.fg_delta_work(_delta(split), 0) > L.fg_delta_work(_delta(long), 0) / 64


def test_refused_steps_norms_and_dropouts():
    L = native.lib()
    step = lambda *n: delta._STEP.pack(*[0] * 26, *n, 1.0)       # noqa: E731  n_slots, batch, heads, three more, dim, value_dim, type
    for n, words in (((4, -1, 2, 2, 2, 2, 64, 64, 0), "negative"), ((4, 4, 3, 2, 3, 3, 64, 64, 0), "multiple"), ((4, 4, 2, 2, 2, 2, 257, 64, 0), "1 to 256"),
                     ((4, 4, 2, 2, 2, 2, 64, 64, 5), "unknown type"), ((4, 4, 2, 2, 2, 2, 64, 64, 0), "null pointer"), ((4, 1 << 27, 2, 2, 2, 2, 64, 64, 0), "2\\^27")):
        assert L.fg_delta_step(step(*n), None) == -1 and re.search(words, _error()), _error()
    norm = lambda rows, dim, typ=0, eps=1e-5, work=(0, 0), p=0, gw=0: layers._NORM.pack(p, p, p, p, 0, 0, gw, 0, rows, dim, dim, dim, typ, eps, *work)   # noqa: E731
    for a, words in ((norm(-1, 8), "rows"), (norm(4, 0), "dim"), (norm(4, 8, 7), "unknown type"), (norm(4, 8, eps=0.0), "eps"), (norm(4, 8), "null pointer")):
        assert L.fg_layer_norm(a, None) == -1 and re.search(words, _error())
        assert L.fg_layer_norm_bwd(a, None) == -1 and re.search(words, _error())
    assert L.fg_layer_norm_bwd(norm(4, 8, p=4096, gw=4096), None) == -1 and "workspace is too small" in _error()
    drop = lambda n, least, typ=0: layers._DROPOUT.pack(0, 0, 0, 0, 0, 0, n, least, typ)   # noqa: E731
    for a, words in ((drop(-1, 0), "n must be"), (drop(5, 65536), "least"), (drop(5, -1), "least"), (drop(5, 0, 9), "unknown type"), (drop(5, 0), "null pointer")):
        assert L.fg_dropout(a, None) == -1 and re.search(words, _error())
    assert L.fg_dropout(drop(0, 0), None) == 0 and L.fg_layer_norm(norm(0, 8), None) == 0


def test_an_eps_that_is_zero_in_fp32_is_refused():
    L = native.lib()
    a = layers._NORM.pack(0, 0, 0, 0, 0, 0, 0, 0, 4, 8, 8, 8, 0, 1e-60, 0, 0)
    for fn in (L.fg_layer_norm, L.fg_layer_norm_bwd):
        assert fn(a, None) == -1 and "eps" in _error()


def test_no_kernel_is_set_up_once_for_all_devices():
    for f in ("fg_delta.cu", "fg_delta_chain.cuh", "fg_delta_grad.cuh", "fg_layers.cu"):
        text = (native.PKG / "csrc" / f).read_text()
        assert "static const bool" not in text and "static bool" not in text, f

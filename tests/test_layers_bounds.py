"""What layer norm's kernels share between warps, and what they ask of a caller's workspace, restated from the source's rules. Without
a GPU."""
import re

import pytest

from flyguy_b200 import layers, native

SOURCE = (native.PKG / "csrc" / "fg_layers.cu").read_text()
# sums that a row group asks for in turn, as numbers of values for `rows` rows at once: the mean; what it lacks and the squares; back, the two
# sums of the gradient
FORWARD, BACK = (lambda rows: [rows, 2 * rows]), (lambda rows: [rows, 2 * rows, 2 * rows])


def _rules():
    """The size of a place in row_sums as the source has it, and what each kernel's calls give for WIDEST."""
    size = re.search(r"room \+ \(turn \^= 1\) \* (.+?);", SOURCE).group(1)
    return size, {k: set(re.findall(r"row_sums<%s, (.+?)>\(" % k, SOURCE)) for k in ("GROUP", "0")}


@pytest.mark.parametrize("kernel, sums, rows, groups", [
    ("k_norm", FORWARD, 1, 1), ("k_norm", FORWARD, 4, 1), ("k_norm_bwd", BACK, 1, 5), ("k_norm_bwd", BACK, 2, 5), ("k_norm_any", FORWARD, 1, 5),
    ("k_norm_any", BACK, 1, 5)], ids=["norm", "norm of 4 rows", "back", "back of 2 rows", "any", "any back"])
@pytest.mark.parametrize("warps", [1, 2, 8, 9, 13, 16])
def test_two_sums_in_a_row_share_no_word(kernel, sums, rows, groups, warps):
    """A block's warps leave their parts of a sum in a place, meet once, and read all of it. Whoever is through may write the next
    sum's parts while others still read, so that one's words have to be others; the one after that comes behind the next barrier."""
    size, calls = _rules()
    env = {"ROWS": rows}
    widest = calls["0" if kernel == "k_norm_any" else "GROUP"]
    room = re.search(r"%s\(const __grid_constant__.*?__shared__ float room\[(.+?)\];" % kernel, SOURCE, re.S).group(1)
    turn, before = 0, set()
    for n in sums(rows) * groups:
        turn ^= 1
        for w in widest:
            at = turn * eval(size, {"N": n, "WIDEST": eval(w, env)})
            words = set(range(at, at + warps * n))
            assert max(words) < eval(room, env), "the place lies in the room"
            assert not words & before, (kernel, n, sorted(words & before)[:4])
        before = words


def _blocks(rows, dim, wide, ring, any_length=64):
    """Blocks that leave sums of a row's length for gw and gb, at most, from the launches' rules: `wide` values a unit, `ring` where
    rows go through it."""
    if dim > 8192:
        return min(rows, any_length)
    if ring:
        return 4 * 148
    units = -(-dim // wide)
    lanes = (8 if units <= (16 if wide > 1 else 32) else 32 if units <= (64 if wide > 1 else 128) else 0)
    if lanes:
        return min(3 * 148, rows)
    per = 1 if wide > 1 and units <= 512 else 16 // wide if wide > 1 else 4 if units <= 2048 else 16
    block = -(-units // (32 * per)) * 32
    return min(rows, 12 * 148, 148 * max(1, 768 // block))


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 65, 443, 2367, 2368, 100_000])
@pytest.mark.parametrize("dim", [1, 8, 63, 64, 517, 1024, 2047, 4096, 8192, 8193, 20_000, 1 << 20, 1 << 24])
def test_sums_over_rows_fit_their_room_and_little_more(rows, dim):
    """What any of the forms writes lies in the workspace, and that is no more than a row of sums each of as many blocks as there can be."""
    room = native.lib().fg_layer_norm_work(layers._NORM.pack(0, 0, 0, 0, 0, 0, 256, 256, rows, dim, dim, dim, 0, 1e-5, 0, 0))
    stats = 3 * rows if dim > 8192 else 0
    forms = [_blocks(rows, dim, wide, ring) for wide in (1, 4, 8) for ring in ((False, True) if rows >= 16 * 148 else (False,))]
    assert room >= 4 * (max(forms) * 2 * dim + stats)
    assert room <= 4 * (min(rows, 64 if dim > 8192 else 12 * 148) * 2 * dim + stats)

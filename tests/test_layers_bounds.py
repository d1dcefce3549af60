"""What layer norm's kernels share between warps, and what they ask of a caller's workspace, restated from the source's rules. Without
a GPU."""
import re

import pytest

from flyguy_b200 import native

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

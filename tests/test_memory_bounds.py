"""What the memory-over-ticks kernels write into a caller's workspace, restated from the launch's rules, against the room that
the library asks for; and what waits for what inside a kernel. Without a GPU."""
import itertools

import pytest

from flyguy_b200 import memory, native

SIZE = {0: 4, 1: 2, 2: 2}


def _plan(typ, total, heads, dim, turned, each):
    """Blocks of queries and keys of a rotation's backward pass with sums of the weights' gradients."""
    unit = 16 // SIZE[typ]
    lanes = 1
    while lanes < dim // (2 * unit):
        lanes *= 2
    blocks = []
    for h in heads:
        per = 1 if each else 256 // lanes
        while per > 1 and (-(-total // per) < 296 or per * (turned // 2) > 2048):
            per //= 2
        blocks.append(max(1, min(-(-total // per), 592 * h // sum(heads))) if h else 0)
    return blocks


@pytest.mark.parametrize("typ", [0, 1])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 64), (1, 8, 16, 4, 128), (128, 128, 16, 4, 128), (64, 1024, 8, 2, 64), (2, 300, 2, 16, 128),
                                  (1, 700, 1, 8, 64), (3, 5, 4, 0, 32)])
def test_sums_of_weight_gradients_fit_their_room(size, typ):
    """Weights absent, frozen, one for all heads or one for each, on either side: every block's sums lie inside the workspace,
    whose first part are the rows' norms."""
    B, T, H, K, D = size
    L, heads, total = native.lib(), (H, K), B * T
    for forms in itertools.product(("none", "frozen", "one", "frozen each", "each"), repeat=2):
        each = any("each" in f for f in forms)
        wanted = [f in ("one", "each") for f in forms]
        w_head = [D if "each" in f else 0 for f in forms]
        fields = [0] * 32 + [256 * (f != "none") for f in forms] + w_head + [256 * x for x in wanted]
        fields += [H, K, B, T, D, D, 256, 0, 0, 0, 8, typ, 0, 1, 1e-6, 1.0, 0, 0]
        room = L.fg_norm_rotate_work(memory._ROTATE.pack(*fields))
        if not any(wanted):
            assert room == 0
            continue
        norms = -(-total * sum(heads) // 4) * 4
        in_units = all(w_head[i] or not wanted[i] or not heads[i] for i in range(2)) and sum(heads) * D * 4 <= 65536 if each else True
        if in_units:                                                        # every block of both sides leaves its sums
            sums = sum(n * (h if each else 1) * D for n, h in zip(_plan(typ, total, heads, D, D, each), heads))
            assert room >= 4 * (norms + sums), (forms, room, 4 * (norms + sums))
        sets = max(h if w else 1 for h, w, x in zip(heads, w_head, wanted) if x)   # sizes and strides of the general form
        assert room >= 4 * (norms + min(256, total) * sets * D), forms

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


# ---- the waits of the tensor-core scan (fg_decay_tc.cuh) ----------------------------------------------------------------
#
# A wait on an mbarrier tells odd phases from even ones only: it may not start before the phase before its own is over, nor find
# that the one after its own is over too. The kernel's roles as lists of steps; a step runs as soon as it can, or never. What one
# role does is a function of what it waits for, so holding a step and running all others as far as they go shows the worst that
# any timing can do.

def _scan_roles(chunks, partial, own_terms, own_out, rounds, parts, stages=True, a_after_b=True, out_in_turn=True):
    """{role: [step]}; steps ("wait", barrier, phase), ("arrive", barrier), ("do", name), ("issue", queue). Queues are roles of their
    own: what the tensor cores and the copies finish, each thread's in order. stages, a_after_b, out_in_turn false: rules without
    which the waits do not hold."""
    warps = ("0", "1")                                                      # two of the eight of a role stand for all
    full = lambda i: ("wait", f"full{i & 1}", i >> 1)                       # noqa: E731
    staged = lambda b, i: ("wait", f"{b}{i & 1}", i >> 1) if stages else ("wait", b, i)   # noqa: E731
    arrive_staged = lambda b, i: ("arrive", f"{b}{i & 1}" if stages else b)   # noqa: E731
    whole = lambda i: not (partial and i == chunks - 1)                     # noqa: E731
    roles = {n: [] for n in ("copies", "loads", "mma", "mma_queue", "ds", "ds_queue", "store", *("ticks" + w for w in warps), *("state" + w for w in warps))}

    def add(role, *steps):
        roles[role] += steps

    last_round = lambda i: rounds * (i + 1) - 1                             # noqa: E731  (of the whole chunks before)
    for i in range(chunks):
        if i >= 2:
            add("copies", staged("kv", i - 2))
            if not parts:
                add("copies", staged("pv", i - 2))
                if not own_out and stages:
                    add("copies", staged("left", i - 2))
                elif not own_out:
                    add("copies", *(("wait", "stored", rounds * (i - 2) + r) for r in range(rounds)))
        add("copies", ("do", f"load{i}"), ("issue", "loads"))
        add("loads", ("do", f"loaded{i}"), ("arrive", f"full{i & 1}"))
        add("ds", full(i), ("wait", "b", i), ("wait", "s", i), ("do", f"dS{i}"), ("issue", "ds_queue"))
        add("ds_queue", ("do", f"dS done{i}"), arrive_staged("kv", i))
        for w in warps:
            me = "state" + w
            if not parts and own_terms and i:
                add(me, ("wait", "qs", i - 1))
            if not parts:
                add(me, ("do", f"copy S{w} {i}"))
            add(me, ("arrive", "s"))
            if not parts:
                add(me, ("wait", "qk" if own_terms else "qs", i))
            if i:
                add(me, staged("kv", i - 1))
            add(me, full(i), ("do", f"fade{w} {i}"), ("arrive", "b"), staged("kv", i), ("do", f"read dS{w} {i}"))
        if parts:
            continue
        add("mma", full(i))
        if i:
            add("mma", staged("pv", i - 1))
            if own_terms and a_after_b:
                add("mma", ("wait", "b", i - 1))
        add("mma", ("do", f"A{i}"), ("issue", "mma_queue"), ("wait", "s", i))
        if i:
            add("mma", ("wait", "read", i - 1))
        add("mma", ("do", f"O1{i}"), ("issue", "mma_queue"), ("wait", "w", i))
        if not whole(i):
            add("mma", ("wait", "b", i))
        add("mma", ("do", f"O2{i}"), ("issue", "mma_queue"))
        add("mma_queue", ("do", f"A done{i}"), ("arrive", "qk"))
        add("mma_queue", ("do", f"O1 done{i}"), ("arrive", "qs"))
        add("mma_queue", ("do", f"O2 done{i}"), arrive_staged("pv", i))
        for w in warps:
            me = "ticks" + w
            add(me, ("wait", "qk", i), ("do", f"W{w} {i}"), ("arrive", "w"), ("wait", "qs", i), staged("pv", i))
            if not whole(i):
                add(me, ("do", f"read out{w} {i}"), ("arrive", "read"))
            elif own_out or rounds > 1:
                for r in range(rounds):
                    if not own_out and r == 0:
                        add(me, staged("kv", i))
                    if rounds * i + r:
                        add(me, ("wait", "stored", rounds * i + r - 1))
                    if r == rounds - 1:
                        add(me, ("do", f"read out{w} {i}"))
                    add(me, ("do", f"put{w} {i}.{r}"))
                    if r == rounds - 1:
                        add(me, ("arrive", "read"))
                    add(me, ("arrive", "ready"))
            else:                                                           # read at once, put over c
                add(me, ("do", f"read out{w} {i}"), ("arrive", "read"), staged("kv", i))
                if i and out_in_turn:
                    add(me, ("wait", "stored", i - 1))
                add(me, ("do", f"put{w} {i}.0"), ("arrive", "ready"))
        if whole(i):
            for r in range(rounds):
                add("store", ("wait", "ready", rounds * i + r), ("do", f"store{i}.{r}"), ("arrive", "stored"))
            if not own_out and stages:
                add("store", arrive_staged("left", i))
    return roles


_TWO = {"b", "s", "w", "read", "ready"}                                     # barriers that all warps of a role arrive at


def _play(roles, hold=None, cap=None):
    """Everything that can run without the step `hold` (role, number) and without barrier cap[0] finishing phase cap[1]: steps done of
    each role, phases over of each barrier, names done."""
    at, arrived, issued, done = dict.fromkeys(roles, 0), {}, {}, set()
    over = lambda b: min(arrived.get(b, 0) // (2 if b in _TWO else 1), cap[1] if cap and cap[0] == b else 1 << 30)   # noqa: E731
    moved = True
    while moved:
        moved = False
        for role, steps in roles.items():
            while at[role] < len(steps) and (role, at[role]) != hold:
                kind, *x = steps[at[role]]
                if kind == "wait" and over(x[0]) <= x[1]:
                    break
                if role in ("loads", "mma_queue", "ds_queue") and at[role] // 2 >= issued.get(role, 0):
                    break
                if kind == "arrive":
                    arrived[x[0]] = arrived.get(x[0], 0) + 1
                elif kind == "issue":
                    issued[x[0]] = issued.get(x[0], 0) + 1
                elif kind == "do":
                    done.add(x[0])
                at[role] += 1
                moved = True
    return at, over, done


def _waits_that_fail(roles):
    at, _, _ = _play(roles)
    bad = [(role, "stuck") for role in roles if at[role] < len(roles[role])]
    for role, steps in roles.items():
        for n, (kind, *x) in enumerate(steps):
            if kind != "wait":
                continue
            bar, phase = x
            if _play(roles, hold=(role, n))[1](bar) > phase + 1:
                bad.append((role, n, bar, phase, "passed by"))
            if phase and _play(roles, cap=(bar, phase - 1))[0][role] >= n and not any(
                    s == ("wait", bar, phase - 1) for s in steps[:n]):
                bad.append((role, n, bar, phase, "early"))
    return bad


def _out_of_order(roles, chunks, own_terms, own_out, rounds, parts):
    """Pairs (first, then) of accesses to one place that some timing turns round."""
    pairs = []
    for i in range(chunks):
        for w in "01":
            if not parts:
                pairs += [(f"O1 done{i - 1}", f"copy S{w} {i}"), (f"copy S{w} {i}", f"O1{i}"), (f"A done{i}", f"fade{w} {i}"),
                          (f"W{w} {i}", f"O2{i}"), (f"read out{w} {i - 1}", f"O1{i}"), (f"read out{w} {i - 1}", f"O2{i}"),
                          (f"O2 done{i}", f"put{w} {i}.0"), (f"O2 done{i}", f"read out{w} {i}")]
                if not own_terms:
                    pairs += [(f"O1 done{i}", f"fade{w} {i}"), (f"dS done{i - 1}", f"copy S{w} {i}")]
                if not own_out:
                    pairs.append((f"dS done{i}", f"put{w} {i}.0"))
                else:
                    pairs.append((f"store{i - 1}.{rounds - 1}", f"put{w} {i}.0"))
                pairs += [(f"put{w} {i}.{r}", f"store{i}.{r}") for r in range(rounds)]
                pairs += [(f"store{i}.{r - 1}", f"put{w} {i}.{r}") for r in range(1, rounds)]
            pairs += [(f"dS done{i - 1}", f"fade{w} {i}"), (f"loaded{i}", f"fade{w} {i}"), (f"fade{w} {i}", f"dS{i}"),
                      (f"dS done{i}", f"read dS{w} {i}"), (f"read dS{w} {i - 1}", f"dS{i}")]
        pairs += [(f"loaded{i}", f"A{i}"), (f"O2 done{i - 1}", f"A{i}"), (f"dS done{i - 2}", f"load{i}"), (f"O2 done{i - 2}", f"load{i}")]
        if not own_out:
            pairs.append((f"store{i - 2}.{rounds - 1}", f"load{i}"))
    where = {step[1]: (role, n) for role, steps in roles.items() for n, step in enumerate(steps) if step[0] == "do"}
    return [(a, b) for a, b in pairs if a in where and b in where and b in _play(roles, hold=where[a])[2]]


# dim and value_dim up to 64 or 128, out in fp32: places of their own for b's terms and for out, rounds of out a chunk
_FORMS = [(True, True, 1, False), (True, True, 2, False), (False, True, 1, False), (False, False, 1, False), (False, False, 2, False),
          (True, True, 1, True), (False, False, 1, True)]


@pytest.mark.parametrize("form", _FORMS)
def test_no_wait_of_the_scan_is_passed_by(form):
    own_terms, own_out, rounds, parts = form
    for chunks in (1, 2, 3, 6):
        for partial in (False, True):
            roles = _scan_roles(chunks, partial, own_terms, own_out, rounds, parts)
            assert not _waits_that_fail(roles), (chunks, partial)
            assert not _out_of_order(roles, chunks, own_terms, own_out, rounds, parts), (chunks, partial)


@pytest.mark.parametrize("rule,form,role", [({"stages": False}, _FORMS[0], "copies"), ({"stages": False}, _FORMS[3], "ticks0"),
                                            ({"stages": False}, _FORMS[5], "copies"), ({"a_after_b": False}, _FORMS[0], "state0"),
                                            ({"out_in_turn": False}, _FORMS[3], "store")])
def test_the_restatement_finds_waits_that_can_be_passed_by(rule, form, role):
    """Without one of the rules, planted here: a wait that another phase can overtake."""
    own_terms, own_out, rounds, parts = form
    found = _waits_that_fail(_scan_roles(6, False, own_terms, own_out, rounds, parts, **rule))
    assert any(f[0] == role and f[-1] == "passed by" for f in found), found

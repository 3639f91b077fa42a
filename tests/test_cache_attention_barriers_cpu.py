"""The order that the barriers of attn_tc_kernel (csrc/cache_attention_tcgen05.cuh) enforce, searched on the CPU through every
interleaving of its roles: a wait goes by a phase's parity alone, so an arrival that may come twice before a waiter has looked
once is a deadlock that no timing shows."""

import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bittorch_b200", "csrc", "cache_attention_tcgen05.cuh")
SLOTS = 4                                                                   # of the ring of key and value tiles


def checked_barriers():
    """How many barriers say that a block's values have been looked through."""
    text = open(SOURCE).read()
    assert int(re.search(r"constexpr int TC_SLOTS = (\d+);", text).group(1)) == SLOTS
    found = re.search(r"uint64_t v_checked(?:\[(\d+)\])?;", text)
    return int(found.group(1) or 1)


def roles(pieces, checked):
    """pieces: (blocks, how many of them at the end hold new tokens) of pairs of tiles that share their keys and values.
    -> programs of ("wait", barrier, phase) / ("arrive", barrier), and how many arrivals complete each barrier's phase.  The
    second stream is two warps; products complete in the order of their issue, at any time after it."""
    tma, scores, outputs = [], [], []
    stream = [[], []]
    counts = {}
    number = {}                                                             # phases that a role has gone through, by barrier and role

    def phase(key):
        number[key] = number.get(key, 0) + 1
        return number[key] - 1

    tile = 0
    unread = None
    fetched = [0, 0]
    for at, (blocks, tails) in enumerate(pieces):
        order = [("k", j) for j in range(min(2, blocks))]
        for j in range(blocks):
            order += [("v", j)] + ([("k", j + 2)] if j + 2 < blocks else [])
        place = {}
        for what in order:
            place[what] = (tile % SLOTS, tile // SLOTS)
            slot, turn = place[what]
            tma += [("wait", ("empty", slot), turn - 1), ("arrive", ("full", slot))]
            tile += 1
        for j in range(blocks):
            slot, turn = place["k", j]
            for x in range(2):
                if x == 0:
                    scores.append(("wait", ("full", slot), turn))
                if j == 0:
                    scores.append(("wait", ("q_full", x), at))
                if unread is not None:
                    scores.append(("wait", ("s_read", unread), phase(("s_read", unread))))
                unread = x
                scores.append(("product", [("s_full", x)] + ([("empty", slot)] if x else [])))
            slot, turn = place["v", j]
            for x in range(2):
                if x == 0:
                    outputs.append(("wait", ("full", slot), turn))
                outputs.append(("wait", ("p_full", x), phase(("p_full", x))))
                outputs.append(("product", [("pv_done", x)] + ([("empty", slot)] if x else [])))
        for x in range(2):
            if fetched[x] == at:
                stream[x].append(("arrive", ("q_full", x)))                 # the first piece's queries
                fetched[x] += 1
            for j in range(blocks):
                stream[x] += [("wait", ("s_full", x), phase(("s_full", x))), ("arrive", ("s_read", x))]
                if j > 0:
                    stream[x].append(("wait", ("pv_done", x), phase(("pv_done", x))))
                if j >= blocks - tails:
                    n = phase(("checked", x))
                    if x == 0:
                        stream[x] += [("wait", ("full", place["v", j][0]), place["v", j][1]), ("arrive", ("v_checked", n % checked))]
                    else:
                        stream[x].append(("wait", ("v_checked", n % checked), n // checked))
                stream[x].append(("arrive", ("p_full", x)))
            if at + 1 < len(pieces):
                stream[x].append(("arrive", ("q_full", x)))
                fetched[x] += 1
            stream[x].append(("wait", ("pv_done", x), phase(("pv_done", x))))
    for name in ("q_full", "s_read", "p_full"):
        counts[name, 1] = 2                                                 # both warps of the second stream
    return [tma, scores, outputs, stream[0], stream[1], stream[1]], counts


def deadlocks(pieces, checked):
    """Whether some interleaving stops before every role has ended.  State: places in the programs, and how many of the
    issued products of the two issuing warps have completed."""
    programs, counts = roles(pieces, checked)
    products = [[op[1] for op in programs[i] if op[0] == "product"] for i in (1, 2)]
    issued = [[0] for _ in range(6)]
    arrivals = []                                                           # per role: arrivals at each barrier before each place
    for i, program in enumerate(programs):
        seen, table = {}, [{}]
        for op in program:
            if op[0] == "arrive":
                seen = dict(seen)
                seen[op[1]] = seen.get(op[1], 0) + 1
            table.append(seen)
            issued[i].append(issued[i][-1] + (op[0] == "product"))
        arrivals.append(table)
    done = []
    for queue in products:
        seen, table = {}, [{}]
        for commits in queue:
            seen = dict(seen)
            for bar in commits:
                seen[bar] = seen.get(bar, 0) + 1
            table.append(seen)
        done.append(table)

    def phases(state, bar):
        n = sum(arrivals[i][state[i]].get(bar, 0) for i in range(6)) + sum(done[i][state[6 + i]].get(bar, 0) for i in range(2))
        return n // counts.get(bar, 1)

    start = (0,) * 8
    todo, known = [start], {start}
    while todo:
        state = todo.pop()
        moves = []
        for i, program in enumerate(programs):
            if state[i] == len(program):
                continue
            op = program[state[i]]
            if op[0] != "wait" or (phases(state, op[1]) & 1) != (op[2] & 1):
                moves.append(state[:i] + (state[i] + 1,) + state[i + 1:])
        for i in range(2):
            if state[6 + i] < issued[1 + i][state[1 + i]]:
                moves.append(state[:6 + i] + (state[6 + i] + 1,) + state[7 + i:])
        if not moves and any(state[i] < len(programs[i]) for i in range(6)):
            return True
        for move in moves:
            if move not in known:
                known.add(move)
                todo.append(move)
    return False


CASES = [[(1, 1)], [(2, 1)], [(2, 2)], [(3, 2)], [(3, 3)], [(4, 2)], [(1, 1), (1, 1)], [(1, 1), (1, 1), (1, 1)], [(2, 1), (1, 1)], [(1, 1), (2, 2)],
         [(2, 2), (2, 1)]]


@pytest.mark.parametrize("pieces", CASES)
def test_no_wait_can_be_lapped(pieces):
    assert not deadlocks(pieces, checked_barriers())


def test_the_search_finds_a_lapped_wait():
    """With one barrier the first stream may arrive for a second block before a warp of the second has looked for the first."""
    assert deadlocks([(3, 2)], 1) and deadlocks([(1, 1), (1, 1), (1, 1)], 1)
    assert not deadlocks([(3, 1)], 1)


def test_every_wait_of_the_kernel_gives_up():
    """A role whose wait runs out leaves for the end of the kernel; whoever waits for it must give up too.  So no wait between
    the CTA's first barrier and its last is one that does not: no barrier by number, no polling without a limit."""
    text = open(SOURCE).read()
    kernel = text[text.index("attn_tc_kernel(const __grid_constant__"):text.index("// Adds up the pieces")]
    assert kernel.count("__syncthreads();") == 2                            # every thread comes to both, whatever it has given up
    assert not re.search(r"bar\.sync|barrier\.(cta\.)?sync|named_barrier", text)
    assert not re.search(r"while\s*\(\s*!\s*mbar_try_wait", text)
    assert set(re.findall(r"\b(\w*wait\w*)\(", kernel)) <= {"wait_or_abort", "wait_or_abort_warp", "mbar_wait_bounded", "tmem_ld_wait", "tmem_st_wait",
                                                             "pdl_wait", "cp_async_wait", "report_wait_timeout"}
    # each wait that gives up is looked at
    for line in kernel.splitlines():
        for found in re.finditer(r"wait_or_abort(_warp)?\(|stream_together\([01]\)", line):
            before = line[:found.start()].rstrip()
            assert before.endswith(("!", "ok = ok &&", "|| !", "return")), line

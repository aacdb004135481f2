"""The waits between the warps of the distillation kernel (ctorch_b200/csrc/losses_held.cu), as a model of one CTA
whose every order of steps is tried: the producer, the copies in flight (which land in any order), the two
list warps, which take turns, and the consumers, which fold `depth` rows ahead of the one that they write.

An mbarrier is a count of completed phases, and a wait with a parity passes when the phase of that parity is not
the open one, as the hardware's test does. The row warp is left out: a coefficient is there as soon as its row is
folded, which allows more orders than the kernel has.
"""
import pytest

LIST_WARPS, SIDES = 2, 8


def passes(completed, parity):
    return completed & 1 != parity


class Fault(Exception):
    pass


def programs(rows, depth, flushes):
    """The steps of each list warp and of the consumers. A row in `flushes` is followed by so many rows that do not
    count that it is written, and its list put, before the next one is taken."""
    lists = []
    for w in range(LIST_WARPS):
        steps, held = [], None
        for row in range(rows):
            if row % LIST_WARPS == w:
                steps.append(("take", row))
                if held is not None:
                    steps.append(("put", held))
                held = row
            if row in flushes and held is not None:
                steps.append(("put", held))
                held = None
        if held is not None:
            steps.append(("put", held))
        lists.append(steps)
    consumer, written = [], 0
    for row in range(rows):
        consumer.append(("fold", row))
        if row - written == depth:
            consumer.append(("write", written))
            written += 1
        if row in flushes:
            while written <= row:
                consumer.append(("write", written))
                written += 1
    while written < rows:
        consumer.append(("write", written))
        written += 1
    return lists, consumer


def explore(rows, stages, depth, flushes, by_row):
    """Tries every order. by_row: `done` has a barrier for each of SIDES rows, and a row is taken only after the row
    before in its stage is written; else `done` belongs to the stage and a list warp waits for its own row alone."""
    lists, consumer = programs(rows, depth, flushes)
    start = (0, frozenset(), (0, 0), 0)  # issued rows, landed rows, steps of the list warps, of the consumers
    seen, todo = {start}, [start]
    while todo:
        issued, landed, at, c = todo.pop()
        folded = sum(s[0] == "fold" for s in consumer[:c])
        written = c - folded
        taken = {s[1] for w in range(LIST_WARPS) for s in lists[w][: at[w]] if s[0] == "take"}
        full = lambda slot: sum(r % stages == slot for r in landed)

        def done(row):
            mine = SIDES if by_row else stages
            return passes(sum(r % mine == row % mine for r in range(written)), row // mine & 1)

        after = []
        if issued < rows and issued - stages < written:
            after.append((issued + 1, landed, at, c))
        for r in range(issued):
            if r not in landed:
                after.append((issued, landed | {r}, at, c))
        for w in range(LIST_WARPS):
            if at[w] == len(lists[w]):
                continue
            what, row = lists[w][at[w]]
            if what == "take":
                free = passes(full(row % stages), row // stages & 1)
                if by_row and row >= stages:
                    free = free and done(row - stages)
                if free and row not in landed:
                    raise Fault(f"row {row} taken before it has landed")
            else:
                free = done(row)
                if free and row >= written:
                    raise Fault(f"row {row} put before it is written")
            if free:
                after.append((issued, landed, tuple(n + (k == w) for k, n in enumerate(at)), c))
        if c < len(consumer):
            what, row = consumer[c]
            if what == "write" or (row in taken and row in landed):
                after.append((issued, landed, at, c + 1))
        if not after and (c < len(consumer) or any(n < len(s) for n, s in zip(at, lists))):
            raise Fault("a wait that nothing ends")
        for s in after:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return len(seen)


@pytest.mark.parametrize("rows,flushes,what", [(4, (), "landed|nothing ends"), (7, (3,), "landed|nothing ends")])
def test_the_model_finds_barriers_by_stage_wrong(rows, flushes, what):
    with pytest.raises(Fault, match=what):
        explore(rows, 3, 1, flushes, by_row=False)


@pytest.mark.parametrize("flushes", [(), (0,), (1,), (2, 3), (3,), (4, 5)])
@pytest.mark.parametrize("stages", [3, 4, 5, 6, 7, 8])
def test_no_order_of_steps_goes_wrong(stages, flushes):
    depth = 3 if stages >= 6 else 2 if stages >= 5 else 1
    for rows in (1, 2, 3, 4, stages + 1, SIDES + 4):
        assert explore(rows, stages, depth, flushes, by_row=True) > rows

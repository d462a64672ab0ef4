"""Copies under way when a wait of the few-rows attention kernel gives up, checked on the CPU.

Two warps load the page boxes of a stream of K and V tiles into a ring of stages; the second skips tiles of a single
box. Before shared memory is released, every copy has to be awaited by somebody: a tile's barrier completes only with
the copies of both warps, but the first warp awaits only the tiles that it has reached itself. This test restates the
order of publishing, loading and freeing, stops it at every moment with the copies as late as they can be, and takes
from the kernel's source who waits and for how many tiles.
"""
import random
import re
from pathlib import Path

SOURCE = (Path(__file__).resolve().parent.parent / "flashlite_b200" / "csrc" / "fl_tree_few.cu").read_text()


def awaited(worker, n, issued, stages):
    """Tiles that the source's last loop has this warp wait for; issued: the tiles it has copies in."""
    at = SOURCE.index("if (*abort_flag && lane == 0")
    block = SOURCE[at:SOURCE.index("S^T = K Q^T ====", at)]
    if "worker == 0" in block[:block.index("\n")] and worker != 0:
        return set()
    span = re.search(r"kUnderWay = kStages \+ (\d+)", block)
    span = stages + int(span.group(1)) if span else stages
    own = "if (issued >>" in block
    return {i for i in range(max(n - span, 0), n) if not own or i in issued}


def stop_at_every_moment(rng, stages, segments):
    """segments: boxes of each tile. Yields (n, issued) of both warps and the copies still under way."""
    tiles = [(s, t, b) for s, boxes in enumerate(segments) for t, b in enumerate(boxes)]
    stream = [entry for entry in tiles for _ in range(2)]  # K and V
    n, issued, landed, freed = [0, 0], [set(), set()], set(), 0
    while True:
        published = stream[n[0]][0] if n[0] < len(stream) else len(segments)
        yield n, issued, landed
        moves = []
        for w in (0, 1):
            if n[w] < len(stream) and stream[n[w]][0] <= published:
                if w == 1 and stream[n[w]][2] <= 1:
                    moves.append(("skip", w))
                elif n[w] - stages < freed:
                    moves.append(("load", w))
        ready = freed < len(stream) and freed in issued[0] and (stream[freed][2] <= 1 or freed in issued[1])
        if ready:
            moves.append(("use", None))
        if not moves:
            assert freed == len(stream)
            return
        kind, w = rng.choice(moves)
        if kind == "skip":
            n[w] += 2 - n[w] % 2
        elif kind == "load":
            issued[w].add(n[w])
            n[w] += 1
        else:  # a tile is used as late as it can be, and its copies land only then
            landed.add(freed)
            freed += 1


def test_every_copy_is_awaited():
    rng = random.Random(0)
    for stages in (3, 6):
        for _ in range(300):
            segments = []
            for _ in range(rng.randint(1, 12)):
                last = rng.choice([1, 1, 2, 5])
                segments.append([8] * rng.choice([0, 0, 1, 3]) + [last])
            for n, issued, landed in stop_at_every_moment(rng, stages, segments):
                under_way = (issued[0] | issued[1]) - landed
                waits = awaited(0, n[0], issued[0], stages) | awaited(1, n[1], issued[1], stages)
                assert under_way <= waits, (stages, segments, under_way - waits)

"""The CTA-pair kernel of the 8-bit products (csrc/tc_gemm_fp8.cuh) when a wait is abandoned, as a model under random schedules: two
producers, the MMA thread, epilogue warps of both CTAs, loads and MMAs that end in their own time.  One role gives up at a random
wait, which stops its CTA; the other CTA's waits run out at any time behind that, at the latest when nothing moves any more.
Nothing that is stored lacks a block or holds another one's sums, and no copy or MMA is under way when the CTAs end.  Without the
rules that the kernel follows (no hand-back and no stores behind an abandoned wait; the MMA thread waits for its last MMA, the
leader for the stages behind it) the model finds such stores and such ends."""
import random
import re

import pytest

from .conftest import PKG_ROOT

SOURCE = (PKG_ROOT / "csrc" / "tc_gemm_fp8.cuh").read_text()
STAGES = int(re.search(r"F8_STAGES = (\d+);", SOURCE).group(1))
WARPS = 2  # of each CTA, in place of eight


class Pair:
    def __init__(self, tiles, steps, rules, rng):
        self.tiles, self.steps, self.blocks, self.rules, self.rng = tiles, steps, tiles * steps, rules, rng
        self.abort = [False, False]
        self.issued = [0, 0]                     # stages that a producer has started to load
        self.loading = []                        # (cta, block)
        self.landed = [set(), set()]
        self.consumed = 0                        # blocks whose MMAs are over
        self.started = 0                         # blocks whose MMAs were issued
        self.free = [0, 0]                       # arrivals on each accumulator
        self.tmem = [[None, None], [None, None]]  # block that an accumulator holds or is being filled with
        self.bad = []
        self.roles = [(c, self.producer(c)) for c in (0, 1)] + [(0, self.mma())] + \
            [(c, self.warp(c)) for c in (0, 1) for _ in range(WARPS)]
        self.waits = {}

    def producer(self, c):
        for b in range(self.blocks):
            if not (yield lambda: b < STAGES + self.consumed):
                return
            self.issued[c] = b + 1
            self.loading.append((c, b))

    def mma(self):
        for b in range(self.blocks):
            if not (yield lambda: b in self.landed[0] and b in self.landed[1]):
                return
            if not (yield lambda: self.free[b % 2] >= (b // 2) * 2 * WARPS):
                return
            for c in (0, 1):
                self.tmem[c][b % 2] = b
            self.started = b + 1

    def warp(self, c):
        gave_up = False
        for t in range(self.tiles):
            sums = []
            for b in range(t * self.steps, (t + 1) * self.steps):
                if not gave_up:
                    gave_up = not (yield lambda: self.consumed > b)
                before = self.tmem[c][b % 2] if self.consumed > b else None
                yield None
                sums.append(before if before == self.tmem[c][b % 2] else None)
                if not (gave_up and self.rules):
                    self.free[b % 2] += 1
            if not (self.rules and self.abort[c]) and sums != list(range(t * self.steps, (t + 1) * self.steps)):
                self.bad.append((c, t))
            if gave_up:
                return

    def run(self, give_up_at):
        live = {}
        for i, (c, role) in enumerate(self.roles):
            live[i] = next(role, "over")
        count = 0
        while True:
            live = {i: w for i, w in live.items() if w != "over"}
            if not live:
                return
            ready = [i for i, w in live.items() if w is None or w()]
            stopped = [i for i, w in live.items() if w is not None and not w() and self.abort[self.roles[i][0]]]
            events = [("role", i, True) for i in ready] + [("role", i, False) for i in stopped] + \
                [("land", x, 0) for x in self.loading] + ([("commit", 0, 0)] if self.consumed < self.started else [])
            count += 1
            if count == give_up_at or any(self.abort) and self.rng.random() < 0.05:  # (further limits at any time)
                waiting = [i for i, w in live.items() if w is not None]
                if waiting:
                    i = self.rng.choice(waiting)
                    self.abort[self.roles[i][0]] = True
                    events = [("role", i, False)]
            if not events:
                i = self.rng.choice(list(live))  # a wait that ran into its limit
                self.abort[self.roles[i][0]] = True
                events = [("role", i, False)]
            what, x, ok = self.rng.choice(events)
            if what == "land":
                self.loading.remove(x)
                self.landed[x[0]].add(x[1])
            elif what == "commit":
                self.consumed += 1
            else:
                try:
                    live[x] = self.roles[x][1].send(ok)
                except StopIteration:
                    live[x] = "over"


    def under_way(self, drain):
        """Copies and MMAs that are not over when both CTAs end."""
        if drain:
            self.consumed = self.started
            for b in range(self.started, max(self.issued)):
                if b < min(self.issued):
                    self.loading = [x for x in self.loading if x[1] != b]  # full: both CTAs' copies
                else:
                    self.loading = []  # never full: the limit, longer than any copy takes
        return len(self.loading) + self.started - self.consumed


def ends(drain, runs=3000):
    rng = random.Random(3)
    busy = 0
    for _ in range(runs):
        pair = Pair(rng.randrange(1, 4), rng.randrange(1, 9), True, rng)
        pair.run(rng.randrange(1, 150))
        assert max(pair.issued) - pair.started <= STAGES  # the barriers' phases tell the stages apart
        busy += pair.under_way(drain) > 0
    return busy


def test_nothing_is_under_way_at_the_end():
    assert ends(True) == 0 and ends(False) > 0


def stores(rules, runs=3000):
    rng = random.Random(1)
    bad = 0
    for _ in range(runs):
        pair = Pair(rng.randrange(1, 4), rng.randrange(1, 9), rules, rng)
        pair.run(rng.randrange(1, 150))
        bad += bool(pair.bad)
    return bad


def test_nothing_unfinished_is_stored():
    assert stores(True) == 0


def test_the_model_finds_stores_without_the_rules():
    assert stores(False) > 0


def test_without_an_abandoned_wait_every_tile_is_stored():
    pair = Pair(3, 7, True, random.Random(2))
    pair.run(-1)
    assert pair.abort == [False, False] and not pair.bad and pair.consumed == 21


@pytest.mark.parametrize("rule", [r"arrive_lane0\(tmem_free_leader0 \+ buf \* 8, sign\)", r"arrive_lane0\(tmem_free_leader0 \+ \(it & 1\) \* 8, sign\)",
                                  r"if \(!live \|\| !whole\) continue;", r"bool mine = lane < rows && whole;",
                                  r"mine = mine && other != 0xffffffffu;"])
def test_the_kernel_follows_the_rules(rule):
    """The places where an epilogue warp hands back an accumulator or stores."""
    assert len(re.findall(rule, SOURCE)) == 1
    assert len(re.findall(r"arrive_lane0\(tmem_free", SOURCE)) == 2


def test_the_kernel_waits_for_what_is_under_way():
    """Behind the MMA loop the drain, behind the cluster barrier the stages, ahead of freeing TMEM."""
    places = [r"report_stages\(\(int\)rank, loaded\);", r"report_stages\(2, \(int\)it\);\s+umma_commit_pair\(&ctl->drain, 1\);[^\n]*\n\s+"
              r"mbar_wait_through\(&ctl->drain, 0\);", r"cluster_sync_all\(\);  // nobody frees", r"if \(done\[0\] != done\[2\]",
              r"tmem_dealloc_pair\("]
    at = [re.search(place, SOURCE).start() for place in places]
    assert at == sorted(at)


def test_the_kernel_for_few_rows_hands_nothing_back_either():
    """The same rule in tc_gemm_fp8_thin.cuh, whose warps leave ahead of their stores."""
    thin = (PKG_ROOT / "csrc" / "tc_gemm_fp8_thin.cuh").read_text()
    signs = [line.split("//")[0].strip() for line in thin.splitlines() if "mbar_arrive(&ctl->tmem_free" in line]
    assert signs == ["if (lane == 0 && ok) mbar_arrive(&ctl->tmem_free[s]);"]
    assert re.search(r"const bool leave = __any_sync\(0xffffffffu, !ok\);\s+if constexpr \(!GATE_UP\) \{\s+if \(leave\) break;", thin)


def test_the_kernel_for_few_rows_waits_whoever_gave_up():
    """Its producer waits for its last copies and its MMA thread for its last MMAs also where their own waits have held: whoever reads
    them may have left."""
    thin = (PKG_ROOT / "csrc" / "tc_gemm_fp8_thin.cuh").read_text()
    loop = re.search(r"\n( *)for \(int i = it > STAGES \? it - STAGES : 0; i < it; \+\+i\) mbar_wait_through\(&ctl->full\[i % STAGES\], "
                     r"\(i / STAGES\) & 1\);", thin)
    drain = re.search(r"\n( *)umma_commit\(&ctl->drain\);[^\n]*\n( *)mbar_wait_through\(&ctl->drain, 0\);", thin)
    role = len(re.search(r"\n( *)int it = 0;", thin).group(1))  # indented like the role's first line: under no condition of its own
    assert [len(g) for g in (loop.group(1), *drain.groups())] == [role] * 3

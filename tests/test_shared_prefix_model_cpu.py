"""Two models of the tensor-core kernel of attention_shared_prefix, checked on the CPU.

``protocol`` steps the roles of one CTA (planner, producer, two issuers, eight
softmax warps) in a random order, with copies and products that land at any later
time, and finds signals that are lost, waits that pass a phase early and orders
that stop.  ``deal`` cuts the work of a call into the CTAs' spans and checks that
every key tile is done once and where the partial outputs lie.  Both follow
csrc/prefix_attention_tc.cu role by role and csrc/prefix_attention.cu:plan_tc;
they model the order of the work, not its values.
"""
import random

import pytest

RING = 4                                   # pieces handed on ahead


class Fault(Exception):
    pass


class Bar:
    """An mbarrier: `count` arrivals complete a phase; a wait names a phase's parity."""

    def __init__(self, name, count):
        self.name, self.count, self.here, self.phase = name, count, 0, 0

    def arrive(self):
        self.here += 1
        if self.here == self.count:
            self.here = 0
            self.phase += 1

    def passes(self, phase):
        return (self.phase & 1) != (phase & 1)


def protocol(pieces, dim, halves, seed, idle_waits=True):
    """Runs `pieces` (key tiles, live warps of each stream) through one CTA in an order
    drawn from `seed`; raises Fault.  idle_waits: warps without rows wait for the product
    before they signal the next one."""
    rng = random.Random(seed)
    ST = (4 if halves else 3) if dim == 64 else 2
    each = 1 if halves else 2              # arrivals that free a stage

    def bars(name, n, count):
        return [Bar(f"{name}[{i}]", count) for i in range(n)]
    q_full, q_empty = Bar("q_full", 1), Bar("q_empty", 2)
    k_full, v_full = bars("k_full", ST, 1), bars("v_full", ST, 1)
    k_empty, v_empty = bars("k_empty", ST, each), bars("v_empty", ST, each)
    s_full, s_empty, p_full, o_done = bars("s_full", 2, 1), bars("s_empty", 2, 4), bars("p_full", 2, 4), bars("o_done", 2, 1)
    half_there, half_read = Bar("half_there", 4), Bar("half_read", 4)
    piece_full, piece_empty = bars("piece_full", RING, 1), bars("piece_empty", RING, 11)
    ring = [None] * RING
    landing = []                           # copies in flight: any order
    products = [[], []]                    # of each issuer: in order

    def tiles_of(c, t, g):
        return (c["tiles"] - ((t - g) & 1) + 1) >> 1 if halves else c["tiles"]

    def key_tile(t, j, g):
        return 2 * j + ((t - g) & 1) if halves else j

    def planner():
        for turn, c in enumerate(pieces + [None]):
            yield piece_empty[turn % RING], turn // RING - 1
            ring[turn % RING] = c
            piece_full[turn % RING].arrive()

    def taken():
        """The pieces of the ring, given back by the caller."""
        turn = 0
        while True:
            yield turn, (piece_full[turn % RING], turn // RING)
            turn += 1

    def producer():
        i = g = 0
        for turn, there in taken():
            yield there
            c = ring[turn % RING]
            if c is None:
                return
            piece_empty[turn % RING].arrive()
            if c["tiles"] == 0:
                continue
            if i > 0:
                yield q_empty, i - 1
            landing.append(q_full.arrive)
            i += 1
            for _ in range(c["tiles"]):
                s, ph = g % ST, g // ST
                yield k_empty[s], ph - 1
                landing.append(k_full[s].arrive)
                yield v_empty[s], ph - 1
                landing.append(v_full[s].arrive)
                g += 1

    def issuer(t):
        i = g = cs = 0
        for turn, there in taken():
            yield there
            c = ring[turn % RING]
            if c is None:
                return
            piece_empty[turn % RING].arrive()
            if c["tiles"] == 0:
                continue
            n = tiles_of(c, t, g)
            tile = [g + key_tile(t, j, g) for j in range(n)]

            def issue_s(j):
                def done(s=tile[j] % ST, last=j == n - 1):
                    s_full[t].arrive()
                    k_empty[s].arrive()
                    if last:
                        q_empty.arrive()
                products[t].append(done)

            def issue_o(j):
                def done(s=tile[j] % ST):
                    o_done[t].arrive()
                    v_empty[s].arrive()
                products[t].append(done)
            yield q_full, i
            if n == 0:
                q_empty.arrive()
            if not halves and t == 1 and not any(c["live"][1]):     # no rows: only the barriers go on
                for j in range(n):
                    s, ph = tile[j] % ST, tile[j] // ST
                    yield k_full[s], ph
                    s_full[t].arrive()
                    k_empty[s].arrive()
                    if j == n - 1:
                        q_empty.arrive()
                    yield p_full[t], cs + j
                    yield v_full[s], ph
                    o_done[t].arrive()
                    v_empty[s].arrive()
            else:
                if n > 0:
                    yield k_full[tile[0] % ST], tile[0] // ST
                    if cs > 0:
                        yield (s_empty if dim == 64 else o_done)[t], cs - 1
                    issue_s(0)
                for j in range(n):
                    yield v_full[tile[j] % ST], tile[j] // ST
                    more = j + 1 < n
                    if more:
                        yield k_full[tile[j + 1] % ST], tile[j + 1] // ST
                    if dim == 64 and more:
                        yield s_empty[t], cs + j
                        issue_s(j + 1)
                    yield p_full[t], cs + j
                    issue_o(j)
                    if dim == 128 and more:
                        yield o_done[t], cs + j
                        issue_s(j + 1)
            i += 1
            g += c["tiles"]
            cs += n

    def softmax(t, w):
        cs = g = ih = 0
        for turn, there in taken():
            yield there
            c = ring[turn % RING]
            if c is None:
                return
            n = tiles_of(c, t, g)
            g += c["tiles"]
            idle = not c["live"][0 if halves else t][w]
            for j in range(n):
                yield s_full[t], cs + j
                if idle and idle_waits and cs + j > 0:
                    yield o_done[t], cs + j - 1
                if dim == 64:
                    s_empty[t].arrive()
                if not idle:
                    yield None             # work
                    if dim == 64 and j > 0:
                        yield o_done[t], cs + j - 1
                    yield None
                p_full[t].arrive()
            cs += n
            if n > 0:
                yield o_done[t], cs - 1
            if halves and c["tiles"] > 0:
                if t == 1:                 # O stays until the first stream has read it
                    half_there.arrive()
                    yield half_read, ih
                else:
                    yield half_there, ih
                    yield None
                    half_read.arrive()
                ih += 1
            piece_empty[turn % RING].arrive()

    roles = {"planner": planner(), "producer": producer(), "issuer 0": issuer(0), "issuer 1": issuer(1)}
    roles.update({f"softmax {t}{w}": softmax(t, w) for t in (0, 1) for w in range(4)})
    speed = {k: rng.choice([1, 1, 3, 10]) for k in roles}
    at = dict.fromkeys(roles)              # what each waits for
    while roles:
        acts = [k for k in roles if at[k] is None or at[k][0].passes(at[k][1]) for _ in range(speed[k])]
        acts += [landing] * len(landing) + [q for q in products if q]
        if not acts:
            raise Fault("stopped: " + ", ".join(f"{k} at {b.name} {ph}" for k, (b, ph) in at.items()))
        a = rng.choice(acts)
        if a is landing:
            landing.pop(rng.randrange(len(landing)))()
        elif isinstance(a, list):
            a.pop(0)()
        else:
            if at[a] is not None and at[a][0].phase != at[a][1] + 1:
                raise Fault(f"{a} passes {at[a][0].name} phase {at[a][1]} at phase {at[a][0].phase}")
            try:
                at[a] = next(roles[a])
            except StopIteration:
                del roles[a], at[a]
    left = [b.name for b in (q_full, q_empty, *k_full, *v_full, *k_empty, *v_empty, *s_full, *s_empty, *p_full, *o_done,
                             half_there, half_read, *piece_full) if b.here]
    if left or landing or products[0] or products[1]:
        raise Fault(f"signals left over: {left}")


def draw_pieces(rng, halves):
    """Pieces without key tiles, pairs of row tiles, single ones, warps without rows."""
    out = []
    for _ in range(rng.randint(1, 9)):
        single = halves or rng.random() < 0.4
        rows = [rng.randint(1, 4) if single else 4, 0 if single else rng.randint(1, 4)]
        out.append(dict(tiles=rng.choice([0, 1, 1, 2, 3, 4, 7]), live=[[w < n for w in range(4)] for n in rows]))
    return out


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("halves", [False, True])
def test_protocol(dim, halves):
    rng = random.Random(dim + halves)
    for seed in range(300):
        protocol(draw_pieces(rng, halves), dim, halves, seed)


@pytest.mark.parametrize("dim", [64, 128])
def test_protocol_model_finds_a_lost_signal(dim):
    """Warps without rows that signal the next product before this one is done.  At
    head_dim 128 they cannot: S(j+1) is not asked for until O += P(j) V is done."""
    rng = random.Random(7)
    faults = 0
    for seed in range(300):
        try:
            protocol(draw_pieces(rng, False), dim, False, seed, idle_waits=False)
        except Fault:
            faults += 1
    assert (faults > 0) == (dim == 64)


# ---------------------------------------------------------------------------
# spans
# ---------------------------------------------------------------------------
PAIR, SINGLE, ENDS, SMS, LEAST = 5, 4, 2, 148, 4


def plan(fold, requests, queries, group, kv_heads, prefix_tiles, cache_tiles):
    tokens = requests * queries if fold else queries
    per_tile = 128 // group
    tiles = -(-tokens // per_tile)
    heads = kv_heads * (1 if fold else requests)
    halves = tiles == 1
    keys = max(prefix_tiles + (0 if fold else cache_tiles), 1)
    steps = (keys + 1) // 2 if halves else keys
    each = PAIR if tiles > 1 else SINGLE
    units, least = (steps + ENDS) * each, min(LEAST, steps) * each
    total = (tiles // 2 * PAIR + tiles % 2 * SINGLE) * (steps + ENDS) * heads
    span = max(-(-total // SMS), least)
    cuts = min(2 * -(-units // span), max(units // least, 1))
    at_least = max(-(-units // cuts), least)
    return dict(fold=fold, tokens=tokens, per_tile=per_tile, halves=halves, least=at_least, slots=-(-units // at_least) + 1,
                ctas=min(SMS, -(-total // least)), requests=requests, kv_heads=kv_heads, prefix_tiles=prefix_tiles)


def deal(tc, q_len, own_len):
    """Walks every CTA's span as next_piece does and checks the pieces."""
    def load(r):
        tokens = tc["tokens"] if tc["fold"] else q_len[r]
        tiles = -(-tokens // tc["per_tile"])
        keys = max(1, tc["prefix_tiles"] + (0 if tc["fold"] else -(-own_len[r] // 128)))
        steps = (keys + 1) // 2 if tc["halves"] else keys
        return tiles >> 1, tiles & 1, steps, (steps + ENDS) * (PAIR * (tiles >> 1) + (SINGLE if tiles & 1 else 0))
    requests = 1 if tc["fold"] else tc["requests"]
    heads = tc["kv_heads"]
    total = sum(load(r)[3] * heads for r in range(requests))
    span = max(-(-total // tc["ctas"]), tc["least"])
    items = {}
    for cta in range(tc["ctas"]):
        pos, end = min(cta * span, total), min(cta * span + span, total)
        req = req0 = 0
        pieces = []
        while pos < end:
            pairs, _, steps, head = load(req)
            while pos - req0 >= head * heads:
                req0 += head * heads
                req += 1
                pairs, _, steps, head = load(req)
            kh, y = divmod(pos - req0, head)
            whole = PAIR * (steps + ENDS)
            pair = min(y // whole, pairs)
            at = y - pair * whole
            each = PAIR if pair < pairs else SINGLE
            units = min((steps + ENDS) * each - at, end - pos)
            a, b = min(steps, -(-at // each)), min(steps, -(-(at + units) // each))
            slot = cta - (pos - at) // span
            pos += units
            if a != b:
                pieces.append((a == 0, b == steps))
                assert 0 <= slot < tc["slots"]
                items.setdefault((req, kh, pair), []).append((a, b, slot, cta))
        # the places of partial outputs: one of an item that begins here and goes on, one of an item that came in
        assert sum(first and not last for first, last in pieces) <= 1
        assert sum(not first for first, _ in pieces) <= 1
    for r in range(requests):
        pairs, single, steps, _ = load(r)
        for kh in range(heads):
            for pair in range(pairs + single):
                parts = sorted(items[r, kh, pair])
                assert parts[0][0] == 0 and parts[-1][1] == steps
                assert all(x[1] == y[0] for x, y in zip(parts, parts[1:]))
                assert [x[2] for x in parts] == list(range(len(parts)))           # no slot left out
                assert [x[3] for x in parts] == [parts[0][3] + s for s in range(len(parts))]   # CTAs in a row


def test_spans():
    rng = random.Random(3)
    for _ in range(2000):
        requests, queries = rng.randint(1, 9), rng.randint(1, 900)
        prefix, cache = rng.randint(0, 300), rng.randint(0, 40)
        fold = rng.random() < 0.4 and prefix > 0
        if prefix + cache == 0:
            continue
        tc = plan(fold, requests, queries, rng.choice([1, 2, 3, 4, 8, 128]), rng.choice([1, 2, 5, 16]), prefix, cache)
        deal(tc, [rng.randint(0, queries) for _ in range(requests)], [rng.randint(0, cache * 128) for _ in range(requests)])

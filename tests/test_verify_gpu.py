"""Verification of drafted tokens against a plain implementation in 64 bits, request by request."""
import math

import numpy as np
import pytest
import torch

import qwen_engine_amd  # noqa: F401

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from qwen_engine_amd.kernels import ops
    ops.load_library()
    return ops


def weights(z, t):
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    top = z.max()
    if top == -np.inf:
        return np.zeros_like(z)
    if top == np.inf:
        e = (z == np.inf).astype(np.float64)
    else:
        e = np.where(z == -np.inf, 0.0, np.exp((z - top) / t))
    return e / e.sum()


def pick(w, u):
    run = np.cumsum(w)
    if not run[-1] > 0:
        return -1
    over = (run > u * run[-1]) & (w > 0)
    return int(np.argmax(over)) if over.any() else int(np.nonzero(w)[0][-1])


def plain(logits, counts, drafts, guess, temperature, accept, draw):
    tokens, accepted = [], []
    row = d = 0
    for r, n in enumerate(counts):
        t = float(temperature[r])
        V = logits.shape[1]
        out = None
        for j in range(n + 1):
            z = logits[row + j]
            if not t > 0:
                z = np.where(np.isnan(z), -np.inf, z)
                best = int(np.argmax(z)) if z.max() > -np.inf else -1
                if j == n or drafts[d + j] != best or best < 0:
                    out = best
                    break
                continue
            p = weights(z, t)
            if j == n:
                out = pick(p, float(draw[r]))
                break
            x = int(drafts[d + j])
            q = np.zeros(V)
            if guess is not None:
                q = weights(guess[d + j], t)
            elif 0 <= x < V:
                q[x] = 1.0
            px, qx = (p[x], q[x]) if 0 <= x < V else (0.0, 1.0)
            if px > 0 and float(accept[d + j]) * qx < px:
                continue
            w = np.maximum(p - q, 0.0)
            out = pick(w if w.sum() > 0 else p, float(draw[r]))
            break
        tokens += [int(v) for v in drafts[d:d + j]] + [out] + [-1] * (n - j)
        accepted.append(j)
        row += n + 1
        d += n
    return tokens, accepted


def case(counts, V, seed, spread=2.0, lookup=False, greedy_every=4):
    g = torch.Generator().manual_seed(seed)
    rows, R = sum(counts) + len(counts), len(counts)
    D = rows - R
    logits = torch.randn(rows, V, generator=g) * spread
    t = 0.4 + torch.rand(R, generator=g)
    t[greedy_every - 1::greedy_every] = 0.0
    drafted = torch.cat([torch.arange(n + 1) < n for n in counts])
    guess = logits[drafted] + torch.randn(D, V, generator=g)
    per = t.repeat_interleave(torch.tensor(counts)).unsqueeze(1)
    noise = torch.rand(D, V, generator=g).clamp(1e-7, 1 - 1e-7)
    drafts = torch.where(per > 0, guess / per.clamp(min=0.1) - (-noise.log()).log(), logits[drafted]).argmax(1) if D else torch.zeros(0)
    return dict(logits=logits, counts=counts, drafts=drafts.int(), guess=None if lookup else guess, temperature=t,
                accept=torch.rand(D, generator=g), draw=torch.rand(R, generator=g))


def first_of(counts):
    return torch.tensor([0] + list(np.cumsum([n + 1 for n in counts])), dtype=torch.int32)


def go(ops, c, **more):
    up = lambda v: None if v is None else v.to(DEV)
    return ops.verify_drafts(up(c["logits"]), first_of(c["counts"]).to(DEV), up(c["drafts"]), up(c["guess"]), up(c["temperature"]),
                             up(c["accept"]), up(c["draw"]), **more)


def check(ops, c):
    tokens, accepted = go(ops, c)
    n = lambda v: None if v is None else v.numpy()
    want = plain(n(c["logits"]), c["counts"], n(c["drafts"]), n(c["guess"]), n(c["temperature"]), n(c["accept"]), n(c["draw"]))
    assert accepted.tolist() == want[1]
    assert tokens.tolist() == want[0]
    return want


@pytest.mark.parametrize("lookup", [False, True])
@pytest.mark.parametrize("V", [1, 2, 63, 257, 4095, 4096, 4097, 20000, 151936])
def test_against_64_bits(ops, V, lookup):
    counts = [3, 0, 1, 5, 2, 0, 4, 7, 1, 1, 0, 2] if V < 100000 else [4, 0, 2, 3]
    want = check(ops, case(counts, V, V, lookup=lookup))
    if 63 <= V < 100000:
        assert len(set(want[1])) > 1


def test_one_request(ops):
    for n in (0, 1, 9):
        check(ops, case([n], 5000, 70 + n))


def test_many_requests(ops):
    counts = [(i * 5 + i // 7) % 6 for i in range(700)]
    check(ops, case(counts, 300, 3))


@pytest.mark.parametrize("lookup", [False, True])
@pytest.mark.parametrize("V,counts", [(262145, [1, 0, 2]), (300001, [2, 0, 1]), (1100003, [1]), (1100003, [0, 2, 1])])
def test_very_wide_vocabularies(ops, V, counts, lookup):
    """More pieces and spans than a wave looks at in one go, in one launch and in several; the tokens lie all over the vocabulary."""
    c = case(counts, V, V % 1000, spread=0.5, lookup=lookup, greedy_every=100)
    tokens = set()
    for u in (0.0, 0.2, 0.45, 0.7, 0.9, 0.999):
        c["draw"] = torch.full((len(counts),), u)
        want = check(ops, c)
        tokens |= {t * 8 // V for t in want[0] if t >= 0}
    assert len(tokens) >= 5
    if not lookup:                                                 # (the draft's distribution is the model's, and a number beyond 1 refuses the drafts: p alone)
        drafted = torch.cat([torch.arange(n + 1) < n for n in counts])
        c["guess"], c["accept"] = c["logits"][drafted].clone(), torch.full_like(c["accept"], 1.5)
        for u in (0.1, 0.6, 0.97):
            c["draw"] = torch.full((len(counts),), u)
            check(ops, c)


@pytest.mark.parametrize("lookup", [False, True])
@pytest.mark.parametrize("offset", [0.0, -300.0, 5e4, 2e9])
def test_temperatures_of_all_sizes(ops, offset, lookup):
    """From the smallest that 32 bits hold, where the largest logit has everything, to the largest, where all that is not masked is alike."""
    temperatures = [1e-45, 1e-38, 1e-20, 1e-8, 1e-5, 1e-3, 0.05, 1.0, 30.0, 1e4, 1e9, 1e30, 1e37, 3e38]
    counts = [2] * len(temperatures)
    c = case(counts, 5003, 17, spread=3.0, lookup=lookup, greedy_every=1000)
    c["logits"] += offset
    masked = torch.rand(c["logits"].shape, generator=torch.Generator().manual_seed(4)) < 0.3
    masked[torch.cat([torch.arange(3) < 2 for _ in counts]).nonzero()[:, 0], c["drafts"].long()] = False
    c["logits"][masked] = -math.inf
    c["temperature"] = torch.tensor(temperatures)
    for seed in range(3):
        c["draw"] = torch.rand(len(counts), generator=torch.Generator().manual_seed(seed))
        check(ops, c)


def test_flat_distributions(ops):
    """Nearly equal weights: as many borders of running sums as tokens."""
    check(ops, case([2, 1, 0, 3, 2, 2, 2, 1], 151936, 8, spread=1e-3, greedy_every=100))


def test_same_distribution_accepts_all(ops):
    """Drafts from the model's own logits stand whatever the numbers are, up to the largest below 1."""
    c = case([4, 2, 3], 9000, 5, greedy_every=100)
    drafted = torch.cat([torch.arange(n + 1) < n for n in c["counts"]])
    c["guess"] = c["logits"][drafted].clone()
    c["accept"].fill_(1 - 2.0 ** -24)
    assert check(ops, c)[1] == [4, 2, 3]


def test_masks(ops):
    """Masked tokens, NaN, infinite logits, rows where nothing or one token is left, in the model's and in the drafts' rows."""
    c = case([2, 2, 2, 2, 2, 2, 2, 2, 1, 0], 5000, 6, greedy_every=100)
    z, q = c["logits"], c["guess"]
    z[0, 1000:] = -math.inf                  # the second half of the vocabulary masked
    z[3] = -math.inf                         # a row where nothing weighs
    z[6, 10:4990] = math.nan
    z[9, [17, 4099]] = math.inf              # two infinite ones share everything
    z[12] = -math.inf
    z[12, 4500] = -3.0                       # one token left
    q[8] = -math.inf                         # the draft's own distribution is empty
    q[10] = math.nan
    q[12, 5:] = -math.inf
    z[24:26] = -3e38                         # finite lowest numbers: all alike
    c["temperature"][9] = 1e-30
    z[26] = math.nan
    z[26, 3] = 2.0
    check(ops, c)
    for t in (0.0, -1.0):
        c["temperature"][:] = t
        check(ops, c)
    c["temperature"][:] = math.inf
    z[9] = 0.0                               # (infinite logits at an infinite temperature have no meaning)
    check(ops, c)


def test_greedy_ties_and_drafts_outside(ops):
    c = case([2, 2, 2, 1], 4200, 9, greedy_every=1)
    z = c["logits"]
    z[0, [40, 4150]] = 50.0                  # equal largest ones, in two spans: the lower index
    z[3, [4150, 4199]] = 50.0
    c["drafts"][0], c["drafts"][2] = 40, 4199
    assert check(ops, c)[1][:2] != [0, 2]
    for bad in (-1, 4200, 2 ** 31 - 1, -2 ** 31):
        for t in (0.0, 0.8):
            for guess in (c["guess"], None):
                d = dict(c, drafts=c["drafts"].clone(), temperature=torch.full((4,), t), guess=guess)
                d["drafts"][1::2] = bad
                check(ops, d)


def test_numbers_at_the_ends(ops):
    c = case([3, 1, 0, 2], 4500, 10, greedy_every=100)
    c["logits"][:, 0] = -math.inf            # the first token weighs nothing, nor the last
    c["logits"][:, -1] = -math.inf
    for u in (0.0, 1 - 2.0 ** -24):
        for a in (0.0, 1 - 2.0 ** -24):
            c["draw"].fill_(u)
            c["accept"].fill_(a)
            check(ops, c)
    # numbers outside [0, 1) still give a token that weighs something
    c["accept"].fill_(math.nan)
    for u in (1.0, 5.0, -1.0, math.nan, math.inf):
        c["draw"].fill_(u)
        tokens, accepted = go(ops, c)
        assert accepted.tolist() == [0, 0, 0, 0]
        first = first_of(c["counts"])[:-1].tolist()
        assert all(0 < tokens[i] < 4499 for i in first)


def test_rows_of_no_request_and_bad_rows(ops):
    """What no request owns stays as it was; a request whose rows are not there is marked, and the others are served."""
    c = case([2, 1, 3], 600, 11)
    want = plain(*(v.numpy() if isinstance(v, torch.Tensor) else v for v in (c["logits"], c["counts"], c["drafts"], c["guess"],
                                                                             c["temperature"], c["accept"], c["draw"])))
    pad = dict(c, logits=torch.cat([c["logits"], torch.zeros(4, 600)]), drafts=torch.cat([c["drafts"], torch.full((4,), 77, dtype=torch.int32)]),
               guess=torch.cat([c["guess"], torch.zeros(4, 600)]), accept=torch.cat([c["accept"], torch.zeros(4)]))
    tokens = torch.full((13,), 99, dtype=torch.int32, device=DEV)
    tokens, accepted = go(ops, pad, tokens=tokens)
    assert tokens.tolist() == want[0] + [99] * 4 and accepted.tolist() == want[1]
    for first, good in (([0, 3, 5, 40], [0, 1]), ([0, 3, 2, 9], [0]), ([-4, 3, 5, 9], [1, 2]), ([0, 3, 5, 5], [0, 1]),
                        ([9, 9, 9, 9], []), ([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0], [])):
        up = lambda v: v.to(DEV)
        tokens = torch.full((9,), 99, dtype=torch.int32, device=DEV)
        tokens, accepted = ops.verify_drafts(up(c["logits"]), up(torch.tensor(first, dtype=torch.int32)), up(c["drafts"]), up(c["guess"]),
                                             up(c["temperature"]), up(c["accept"]), up(c["draw"]), tokens=tokens)
        got = accepted.tolist()
        for r in good:
            assert got[r] == want[1][r], (first, r)
        if not good:
            assert got == [-1, -1, -1] and (tokens == 99).all()


@pytest.mark.parametrize("R,V", [(6, 600), (6, 200003), (400, 300), (1300, 40)])
@pytest.mark.parametrize("lookup", [False, True])
def test_first_rows_that_fall(ops, R, V, lookup):
    """first[] that falls or stands still somewhere: a request whose rows, or whose drafts' rows, are not behind all earlier ones' is marked
    and nothing of it written; every other one gets the tokens that its own rows and temperature give, in one launch and in several."""
    g = np.random.default_rng(R + V)
    counts = [int(v) for v in g.integers(0, 4, R)]
    c = case(counts, V, R, lookup=lookup, greedy_every=2)
    n = lambda v: None if v is None else v.numpy()
    z, d, q, t, a, u = (n(c[k]) for k in ("logits", "drafts", "guess", "temperature", "accept", "draw"))
    rows, starts = len(z), first_of(counts).tolist()
    lists = [[0, 3, 2] + starts[3:], starts[:3] + [starts[2]] + starts[4:], starts[:-1] + [starts[-3]]]
    for _ in range(4):
        bad = list(starts)
        for k in g.integers(0, R + 1, max(1, R // 100)):
            bad[k] = int(g.integers(-2, rows + 3))
        lists.append(bad)
    marked = served = 0
    for first in lists:
        tokens = torch.full((rows,), 99, dtype=torch.int32, device=DEV)
        up = lambda v: None if v is None else v.to(DEV)
        tokens, accepted = ops.verify_drafts(up(c["logits"]), torch.tensor(first, dtype=torch.int32, device=DEV), up(c["drafts"]), up(c["guess"]),
                                             up(c["temperature"]), up(c["accept"]), up(c["draw"]), tokens=tokens)
        want, kept = [99] * rows, []
        for r, (lo, hi) in enumerate(zip(first, first[1:])):
            if not (hi > lo >= r and hi <= rows and hi - 1 - r <= rows - R and all(first[k] - k <= lo - r for k in range(r))):
                kept.append(-1)
                continue
            m = hi - lo - 1
            here = slice(lo - r, lo - r + m)
            got = plain(z[lo:hi], [m], d[here], None if q is None else q[here], t[r:r + 1], a[here], u[r:r + 1])
            want[lo:hi] = got[0]
            kept += got[1]
        marked, served = marked + kept.count(-1), served + len(kept) - kept.count(-1)
        assert accepted.tolist() == kept, first[:8]
        assert tokens.tolist() == want, first[:8]
    assert marked and served


def full(c):
    """The requests of a case over and over, with numbers of their own, until there are so many that acceptance, sums and draw are launches of
    their own (more than 320 spans of 4096 logits)."""
    times = 321 // (len(c["counts"]) * -(-c["logits"].shape[1] // 4096)) + 1
    g = torch.Generator().manual_seed(77)
    d = {k: v * times if k == "counts" else v if v is None else v.repeat(times, *[1] * (v.dim() - 1)) for k, v in c.items()}
    for k in ("accept", "draw"):
        d[k][len(c[k]):] = torch.rand(len(d[k]) - len(c[k]), generator=g)
    return d


@pytest.mark.parametrize("lookup", [False, True])
def test_masks_in_a_full_batch(ops, lookup):
    """The masks, NaN and infinities of test_masks, and rows where nothing weighs, in the launches of a full batch."""
    c = case([2, 2, 2, 2, 2, 2, 2, 2, 1, 0], 5000, 6, greedy_every=100, lookup=lookup)
    z, q = c["logits"], c["guess"]
    z[0, 1000:] = -math.inf
    z[3] = -math.inf
    z[6, 10:4990] = math.nan
    z[9, [17, 4099]] = math.inf
    z[12] = -math.inf
    z[12, 4500] = -3.0
    if q is not None:
        q[8] = -math.inf
        q[10] = math.nan
        q[12, 5:] = -math.inf
    z[24:26] = -3e38
    c["temperature"][9] = 1e-30
    z[26] = math.nan
    z[26, 3] = 2.0
    check(ops, full(c))
    for t in (0.0, -1.0):
        c["temperature"][:] = t
        check(ops, full(c))
    c["temperature"][:] = math.inf
    z[9] = 0.0
    check(ops, full(c))


@pytest.mark.parametrize("lookup", [False, True])
@pytest.mark.parametrize("offset", [0.0, -300.0, 5e4, 2e9])
def test_temperatures_of_all_sizes_in_a_full_batch(ops, offset, lookup):
    temperatures = [1e-45, 1e-38, 1e-20, 1e-8, 1e-5, 1e-3, 0.05, 1.0, 30.0, 1e4, 1e9, 1e30, 1e37, 3e38]
    counts = [2] * len(temperatures)
    c = case(counts, 5003, 17, spread=3.0, lookup=lookup, greedy_every=1000)
    c["logits"] += offset
    masked = torch.rand(c["logits"].shape, generator=torch.Generator().manual_seed(4)) < 0.3
    masked[torch.cat([torch.arange(3) < 2 for _ in counts]).nonzero()[:, 0], c["drafts"].long()] = False
    c["logits"][masked] = -math.inf
    c["temperature"] = torch.tensor(temperatures)
    check(ops, full(c))


def test_flat_distributions_in_a_full_batch(ops):
    check(ops, case([2, 1, 0, 3, 2, 2, 2, 1, 1], 151936, 8, spread=1e-3, greedy_every=100))


def test_ties_and_drafts_outside_in_a_full_batch(ops):
    c = case([2, 2, 2, 1], 4200, 9, greedy_every=1)
    z = c["logits"]
    z[0, [40, 4150]] = 50.0
    z[3, [4150, 4199]] = 50.0
    c["drafts"][0], c["drafts"][2] = 40, 4199
    check(ops, full(c))
    for bad in (-1, 4200, 2 ** 31 - 1, -2 ** 31):
        for t in (0.0, 0.8):
            for guess in (c["guess"], None):
                d = dict(c, drafts=c["drafts"].clone(), temperature=torch.full((4,), t), guess=guess)
                d["drafts"][1::2] = bad
                check(ops, full(d))


def test_numbers_at_the_ends_in_a_full_batch(ops):
    c = full(case([3, 1, 0, 2], 4500, 10, greedy_every=100))
    c["logits"][:, 0] = -math.inf
    c["logits"][:, -1] = -math.inf
    for u in (0.0, 1 - 2.0 ** -24):
        for a in (0.0, 1 - 2.0 ** -24):
            c["draw"].fill_(u)
            c["accept"].fill_(a)
            check(ops, c)
    c["accept"].fill_(math.nan)
    first = first_of(c["counts"])[:-1].long().to(DEV)
    for u in (1.0, 5.0, -1.0, math.nan, math.inf):
        c["draw"].fill_(u)
        tokens, accepted = go(ops, c)
        assert (accepted == 0).all() and ((tokens[first] > 0) & (tokens[first] < 4499)).all()


@pytest.mark.parametrize("batch", [False, True])
@pytest.mark.parametrize("lookup", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_many_drafts(ops, temperature, lookup, batch):
    """More drafts than a block has waves: the first that is refused among the first 16, the last of them, the first behind them, later, and none."""
    counts = [15, 16, 17, 40, 40, 40, 40, 40, 33, 32, 1]
    refused = [15, 15, 16, 14, 15, 16, 31, 32, 33, 7, 0]           # (as many as there are drafts: none)
    c = case(counts, 700, 60, lookup=lookup, greedy_every=1000)
    c["temperature"].fill_(temperature)
    row = d = 0
    for n, r in zip(counts, refused):
        c["drafts"][d:d + n] = c["logits"][row:row + n].argmax(1)
        c["accept"][d:d + n] = 0.0
        if r < n:
            c["accept"][d + r:d + n] = 1e30
            c["drafts"][d + r] = (c["drafts"][d + r] + 1) % 700
        row, d = row + n + 1, d + n
    if batch:                                                      # (behind one another as they are: the numbers decide)
        c = {k: v * 30 if k == "counts" else v if v is None else v.repeat(30, *[1] * (v.dim() - 1)) for k, v in c.items()}
        refused = refused * 30
    assert check(ops, c)[1] == refused


def test_rows_of_no_request_in_a_full_batch(ops):
    c = full(case([2, 1, 3], 600, 11))
    rows, D = len(c["logits"]), len(c["drafts"])
    want = plain(*(v.numpy() if isinstance(v, torch.Tensor) else v for v in (c["logits"], c["counts"], c["drafts"], c["guess"],
                                                                             c["temperature"], c["accept"], c["draw"])))
    pad = dict(c, logits=torch.cat([c["logits"], torch.zeros(4, 600)]), drafts=torch.cat([c["drafts"], torch.full((4,), 77, dtype=torch.int32)]),
               guess=torch.cat([c["guess"], torch.zeros(4, 600)]), accept=torch.cat([c["accept"], torch.zeros(4)]))
    tokens = torch.full((rows + 4,), 99, dtype=torch.int32, device=DEV)
    tokens, accepted = go(ops, pad, tokens=tokens)
    assert tokens.tolist() == want[0] + [99] * 4 and accepted.tolist() == want[1] and D


def test_recorded_and_two_streams_in_a_full_batch(ops):
    """Recorded twice and replayed on other numbers, with eager work between; then overlapping calls on two streams."""
    cs = [full(case([2, 0, 4, 1], 9001, 20 + i)) for i in range(3)]
    names = ("logits", "drafts", "guess", "temperature", "accept", "draw")
    held = [{k: c[k].to(DEV) for k in names} for c in cs]
    first = first_of(cs[0]["counts"]).to(DEV)

    def run(s):
        return ops.verify_drafts(s["logits"], first, s["drafts"], s["guess"], s["temperature"], s["accept"], s["draw"])

    want = [run(h) for h in held]
    assert want[0][1].tolist() == check(ops, cs[0])[1]
    static = {k: v.clone() for k, v in held[0].items()}
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(static)
        graphs.append((graph, out))
    for _ in range(2):
        for h, w in zip(held, want):
            for k in names:
                static[k].copy_(h[k])
            for graph, out in graphs:
                graph.replay()
            run(held[1])
            torch.cuda.synchronize()
            for graph, out in graphs:
                assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(held[i]))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(t, w[0]) and torch.equal(a, w[1]) for t, a in g)


def test_no_requests(ops):
    e = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device=DEV)
    tokens, accepted = ops.verify_drafts(e(0, 50), torch.zeros(1, dtype=torch.int32, device=DEV), e(0, dtype=torch.int32), None, e(0), e(0), e(0))
    assert tokens.shape == (0,) and accepted.shape == (0,)


def test_logits_beyond_32_bits(ops):
    """More than 2^31 logits: the last requests' tokens are those that they get alone."""
    R, V = 14200, 151936
    g = torch.Generator(device=DEV).manual_seed(2)
    z = torch.randn(R, V, device=DEV, generator=g)
    t = torch.tensor([0.0, 0.9], device=DEV).repeat(R // 2)
    u = torch.rand(R, device=DEV, generator=g)
    none = torch.empty(0, device=DEV)
    first = torch.arange(R + 1, dtype=torch.int32, device=DEV)
    tokens, accepted = ops.verify_drafts(z, first, none.int(), None, t, none, u)
    assert (accepted == 0).all()
    assert torch.equal(tokens[::2].long(), z[::2].argmax(1))
    few, _ = ops.verify_drafts(z[-6:], first[:7], none.int(), None, t[-6:], none, u[-6:])
    assert torch.equal(tokens[-6:], few)


def test_two_streams_at_once(ops):
    """Calls on two streams that overlap do not share anything."""
    cs = [case([3, 1, 2, 4], 30000, 40 + i) for i in range(2)]
    want = [tuple(v.tolist() for v in go(ops, c)) for c in cs]
    up = lambda c: [c[k].to(DEV) for k in ("logits", "drafts", "guess", "temperature", "accept", "draw")] + [first_of(c["counts"]).to(DEV)]
    held = [up(c) for c in cs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cs], [[], []]
    for _ in range(20):
        for i, (s, (z, d, q, t, a, u, f)) in enumerate(zip(streams, held)):
            with torch.cuda.stream(s):
                got[i].append(ops.verify_drafts(z, f, d, q, t, a, u))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all((tokens.tolist(), accepted.tolist()) == w for tokens, accepted in g)


@pytest.mark.parametrize("lookup", [False, True])
def test_tokens_are_distributed_as_the_models(ops, lookup):
    """20 000 requests with one draft each from another distribution: the first token's frequencies are the model's.  A count of n
    trials with probability p is within 5 sqrt(n p (1 - p)) + 5 of n p but once in a million."""
    R, V = 20000, 12
    g = torch.Generator().manual_seed(1)
    p_row, q_row = torch.randn(V, generator=g) * 1.5, torch.randn(V, generator=g)
    q = torch.softmax(q_row.double(), 0)
    drafts = torch.multinomial(q, R, replacement=True, generator=g).int() if not lookup else torch.randint(0, 3, (R,), generator=g).int()
    rows = p_row.repeat(2 * R, 1)
    first = torch.arange(0, 2 * R + 1, 2, dtype=torch.int32)
    tokens, _ = ops.verify_drafts(rows.to(DEV), first.to(DEV), drafts.to(DEV), None if lookup else q_row.repeat(R, 1).to(DEV),
                                  torch.ones(R, device=DEV), torch.rand(R, generator=g).to(DEV), torch.rand(R, generator=g).to(DEV))
    counts = torch.bincount(tokens[::2].cpu().long(), minlength=V).double()
    p = torch.softmax(p_row.double(), 0)
    assert ((counts - R * p).abs() <= 5 * (R * p * (1 - p)).sqrt() + 5).all()


def test_recorded_and_on_another_stream(ops):
    cs = [case([2, 0, 4, 1], 9001, 20 + i) for i in range(4)]
    up = lambda v: v.to(DEV)
    names = ("logits", "drafts", "guess", "temperature", "accept", "draw")
    static = {k: up(cs[0][k]).clone() for k in names}
    first = first_of([2, 0, 4, 1]).to(DEV)

    def run(s):
        return ops.verify_drafts(s["logits"], first, s["drafts"], s["guess"], s["temperature"], s["accept"], s["draw"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alone = run(static)
    torch.cuda.current_stream().wait_stream(side)
    want = [run({k: up(c[k]) for k in names}) for c in cs]
    assert torch.equal(alone[0], want[0][0]) and torch.equal(alone[1], want[0][1])
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(static)
        graphs.append((graph, out))
    for _ in range(2):
        for c, w in zip(cs, want):
            for k in names:
                static[k].copy_(up(c[k]))
            for graph, out in graphs:
                graph.replay()
            run({k: up(cs[1][k]) for k in names})
            torch.cuda.synchronize()
            for graph, out in graphs:
                assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])


def test_sampler_verify(ops):
    from qwen_engine_amd.sampling.sampler import Sampler
    c = case([2, 0, 3], 700, 30)
    flat, acc = c["drafts"].tolist(), c["accept"].tolist()
    drafts, accept = [flat[:2], [], flat[2:]], [acc[:2], [], acc[2:]]
    got = Sampler().verify(c["logits"].to(DEV), drafts, c["guess"].to(DEV), c["temperature"].tolist(), accept, c["draw"].tolist())
    tokens, accepted = go(ops, c)
    tokens, accepted = tokens.tolist(), accepted.tolist()
    want = [tokens[lo:lo + n + 1] for lo, n in zip((0, 3, 4), accepted)]
    assert got == want
    assert Sampler().verify(torch.empty(0, 700, device=DEV), [], None, [], [], []) == []
    with pytest.raises(ValueError):
        Sampler().verify(c["logits"].to(DEV), drafts, None, [1.0, 1.0], accept, [0.5, 0.5, 0.5])
    with pytest.raises(ValueError):
        Sampler().verify(c["logits"].to(DEV), [[1], [], [2]], None, [1.0] * 3, [[0.1], [], [0.1]], [0.5] * 3)


def test_drafting_with_a_4_bit_copy(ops):
    """The operators together: a small model's matrices in 4 bits draft tokens that its own matrices verify; at temperature 0
    the tokens are those of the model alone, whatever the copy proposes, and some drafts stand."""
    from qwen_engine_amd.sampling.sampler import Sampler, uniform_for
    g = torch.Generator().manual_seed(4)
    V, H, I, R, n = 500, 128, 256, 3, 4
    table, up, down, head = (torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV) * k
                             for s, k in (((V, H), 1.0), ((2 * I, H), 0.15), ((H, I), 0.15), ((V, H), 0.3)))
    held = {k: ops.mxfp4_quantize(w.contiguous()) for k, w in (("up", up), ("down", down), ("head", head))}

    def model(ids, four):
        h = ops.embedding(torch.tensor(ids, dtype=torch.int32, device=DEV), table)
        x = h.to(torch.bfloat16)
        if four:
            y = ops.gemm_mxfp4(x, held["up"], epilogue=ops.EPI_SILU_MUL)
            ops.gemm_mxfp4(y, held["down"], out=h, epilogue=ops.EPI_RESIDUAL)
            return ops.gemm_mxfp4(h.to(torch.bfloat16), held["head"], out_dtype=torch.float32)
        y = ops.silu_mul(ops.gemm(x, up))
        ops.residual_add(h, ops.gemm(y, down))
        return ops.gemm(h.to(torch.bfloat16), head, out_dtype=torch.float32)

    sampler = Sampler()

    def run(temperatures, steps):
        out, stood = [[5 + r] for r in range(R)], 0
        for _ in range(steps):
            drafts, rows = [[] for _ in range(R)], []
            last = [o[-1] for o in out]
            for j in range(n):
                z = model(last, True)
                rows.append(z)
                last = sampler.sample(z, temperatures, [uniform_for(1, r, len(out[r]) + j) for r in range(R)])
                for r in range(R):
                    drafts[r].append(last[r])
            logits = model([t for r in range(R) for t in [out[r][-1]] + drafts[r]], False)
            guess = torch.stack(rows, 1).reshape(R * n, V)
            accept = [[uniform_for(1, r, len(out[r]) + j, "accept") for j in range(n)] for r in range(R)]
            got = sampler.verify(logits, drafts, guess, temperatures, accept, [uniform_for(1, r, len(out[r]), "draw") for r in range(R)])
            stood += sum(len(t) - 1 for t in got)
            for r in range(R):
                out[r] += got[r]
        return out, stood

    out, stood = run([0.0] * R, 6)
    assert stood > 0
    for o in out:
        for a, b in zip(o, o[1:]):
            z = model([a], False)
            row = z[0].double().cpu()
            # (the verifying step multiplies more rows at a time: a near tie may fall the other way)
            assert float(row.max() - row[b]) <= 2e-2 * float(row.abs().max())
    out, stood = run([0.8, 0.0, 1.2], 6)
    assert stood > 0 and all(0 <= t < V for o in out for t in o)

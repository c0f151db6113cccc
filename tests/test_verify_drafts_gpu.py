"""Verification of drafted tokens against the rule in float64, request by request, and against the distribution it has to give."""

from __future__ import annotations

import struct

import pytest
import torch

import miniserve_b200  # noqa: F401
from miniserve_b200 import kernels
from miniserve_b200.kernels import KernelError

pytestmark = pytest.mark.gpu


def records_of(settings):
    """int32 [slots, 8] of (temperature, top_p, top_k) each."""
    return torch.tensor([struct.unpack("<8i", struct.pack("<ffiIIiii", t, p, k, 7, 0, 0, 0, 0)) for t, p, k in settings], dtype=torch.int32).cuda()


def make(drafts, vocab, settings, probabilities, seed=0, spread=3.0, grid=None):
    """``grid``: logits are multiples of it (equal ones are then common)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    count, total = len(drafts), sum(drafts)
    rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")
    logits = spread * torch.randn(total + count, vocab, generator=g, device="cuda")
    if grid:
        logits = torch.round(logits / grid) * grid
    starts = [0]
    for d in drafts:
        starts.append(starts[-1] + d)
    rows = [starts[r] + r + i for r in range(count) for i in range(drafts[r])]
    near = torch.softmax(logits[rows] + 0.5 * torch.randn(total, vocab, generator=g, device="cuda"), -1)
    chosen = (near / torch.empty_like(near).exponential_(generator=g)).argmax(-1) if total else torch.zeros(0)
    if not probabilities and total:
        chosen = torch.where(rand(total) < 0.6, logits[rows].argmax(-1), chosen)
    ints = lambda values: torch.tensor(values, dtype=torch.int32).cuda()
    slots = [(5 * r + 3) % (count + 1) for r in range(count)] if (count + 1) % 5 else list(range(count))
    table = [(0.5, 0.5, 3)] * (count + 1)
    for r, slot in enumerate(slots):
        table[slot] = settings[r % len(settings)]
    return dict(logits=logits, drafts=chosen.int().cuda(), draft_start=ints(starts), uniforms=rand(total),
                noise=torch.empty(count, vocab, device="cuda").exponential_(generator=g), draft_probs=near if probabilities else None,
                records=records_of(table), slot_of_request=ints(slots), settings=[settings[r % len(settings)] for r in range(count)])


def verify(case, with_probs=True):
    count, total = case["draft_start"].numel() - 1, case["drafts"].numel()
    accepted, token = (torch.full((count,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    target = torch.full((total,), -9.0, device="cuda") if with_probs else None
    kernels.verify_drafts(case["logits"], case["drafts"], case["draft_start"], case["uniforms"], case["noise"], accepted, token,
                          draft_probs=case["draft_probs"], records=case["records"], slot_of_request=case["slot_of_request"], target_probs=target)
    return accepted, token, target


def distribution(row, setting):
    """The kept tokens' probabilities in float64."""
    temperature, top_p, top_k = setting
    top_p = struct.unpack("f", struct.pack("f", top_p))[0]
    temperature = struct.unpack("f", struct.pack("f", temperature))[0]
    x = torch.nan_to_num(row.double(), nan=-float("inf"), posinf=float("inf"), neginf=-float("inf"))
    p = torch.zeros_like(x)
    top = x.max()
    if top == -float("inf"):
        return p
    if temperature == 0.0:
        p[int(x.argmax())] = 1.0
        return p
    if top == float("inf"):
        p = (x == top).double()
    else:
        p = torch.exp((x - top) / temperature)
    order = torch.sort(x, descending=True, stable=True).indices
    if 0 < top_k < len(x):
        p[order[top_k:]] = 0.0
    if top_p < 1.0:
        mass = p[order]
        p[order[mass.cumsum(-1) - mass > top_p * mass.sum()]] = 0.0
    return p / p.sum()


def expected(case):
    starts, drafts = case["draft_start"].tolist(), case["drafts"].tolist()
    accepted, tokens, target = [], [], []
    for r, setting in enumerate(case["settings"]):
        row, taken, source = starts[r] + r, 0, None
        for i in range(starts[r], starts[r + 1]):
            p = distribution(case["logits"][row + i - starts[r]], setting)
            inside = 0 <= drafts[i] < len(p)
            target.append(float(p[drafts[i]]) if inside else 0.0)
            if source is not None:
                continue
            if case["draft_probs"] is not None:
                q = case["draft_probs"][i].double()
            else:
                q = torch.zeros_like(p)
                if inside:
                    q[drafts[i]] = 1.0
            passes = target[-1] > 0.0 if setting[0] == 0.0 else float(case["uniforms"][i]) * (float(q[drafts[i]]) if inside else 1.0) < target[-1]
            if passes:
                taken += 1
            else:
                less = (p - q).clamp(min=0.0)
                source = p if setting[0] == 0.0 or not bool((less > 0).any()) else less
        if source is None:
            source = distribution(case["logits"][row + taken], setting)
        accepted.append(taken)
        if not bool((source > 0).any()):
            tokens.append(0)
        else:
            tokens.append(int((source if setting[0] == 0.0 else torch.where(source > 0, source / case["noise"][r].double(), -1.0)).argmax()))
    return accepted, tokens, target


def check(case):
    accepted, token, target = verify(case)
    want = expected(case)
    assert accepted.tolist() == want[0]
    assert token.tolist() == want[1]
    # p: an exponential of an argument that is off by 2^-23 of itself (up to |ln p| <= 104) and 2 ulp, over a sum of the same: 2 (104 2^-23 + 2^-21)
    for got, p in zip(target.tolist(), want[2]):
        assert abs(got - p) <= p * 2 * (104 * 2.0 ** -23 + 2.0 ** -21) + 1e-37
    again = verify(case)
    assert torch.equal(again[0], accepted) and torch.equal(again[1], token) and torch.equal(again[2], target)


PLAIN, GREEDY = (0.8, 1.0, 0), (0.0, 1.0, 0)


@pytest.mark.parametrize("probabilities", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 7, 33, 500, 4096, 32011, 151936])
def test_without_filters(vocab, probabilities):
    check(make([3, 0, 5, 1, 2, 8, 1], vocab, [PLAIN, GREEDY, (1.5, 1.0, vocab), (0.3, 1.0, 0)], probabilities, seed=vocab))


@pytest.mark.parametrize("probabilities", [True, False])
@pytest.mark.parametrize("vocab", [2, 7, 33, 500, 4096, 32011, 151936])
@pytest.mark.parametrize("settings", [[(1.0, 0.9, 0), (0.7, 0.3, 0), (1.3, 0.999, 0)], [(1.0, 1.0, 1), (0.7, 1.0, 5), (1.3, 1.0, 300)],
                                      [(1.0, 0.9, 20), (0.7, 0.5, 2), (1.3, 0.97, 400), (0.0, 0.5, 3), (1.0, 1e-6, 0)]])
def test_filters(vocab, probabilities, settings):
    check(make([3, 0, 5, 1, 2], vocab, settings, probabilities, seed=vocab + len(settings)))


@pytest.mark.parametrize("count,vocab", [(64, 33001), (140, 33001), (140, 700), (512, 300), (513, 300)])
@pytest.mark.parametrize("settings", [[(1.0, 0.9, 0), (0.0, 1.0, 0), (0.7, 1.0, 20), (1.0, 1.0, 0), (1.2, 0.95, 290)], [(1.0, 0.9, 0)], [(1.0, 1.0, 0), (1.0, 0.9, 3)]])
def test_more_rows_than_run_at_once(count, vocab, settings):
    """Rows are then worked at in another order than theirs; neighbouring requests differ in number of drafts and in filters."""
    check(make([(7 * i) % 9 % 6 for i in range(count)], vocab, settings, count % 2 == 0, seed=count))


@pytest.mark.parametrize("vocab", [33, 5000, 32011])
@pytest.mark.parametrize("settings", [[(1.0, 1.0, 7), (1.0, 1.0, 200), (0.5, 1.0, 31)], [(1.0, 0.9, 0), (1.0, 0.5, 0), (0.7, 0.2, 0)],
                                      [(1.0, 0.9, 100), (2.0, 0.6, 20), GREEDY]])
@pytest.mark.parametrize("grid", [0.5, 4.0, 100.0])
def test_equal_logits(vocab, settings, grid):
    """Logits of few values (0.5 apart, 4 apart, all equal): at a border the lower indices stay, an argmax is the first."""
    check(make([3, 2, 0, 4], vocab, settings, True, seed=vocab, grid=grid))


@pytest.mark.parametrize("setting", [PLAIN, GREEDY, (1.0, 0.9, 0), (1.0, 1.0, 3), (0.7, 0.8, 50)])
def test_masked_and_unusual_logits(setting):
    """Rows with -inf for most or all tokens, with NaN, with +inf, with the lowest numbers, of one value, and with zeros of both signs."""
    case = make([4, 4, 3], 1000, [setting], False, seed=3)
    x = case["logits"]
    x[0, 5:] = -float("inf")
    x[1] = -float("inf")
    x[2, ::3] = float("nan")
    x[3, 17] = float("inf")
    x[4] = torch.finfo(torch.float32).min
    x[5] = 0.0
    x[5, ::2] = -0.0
    x[6, 100:] = torch.finfo(torch.float32).min
    x[7] = float("nan")
    x[8, 3] = 1e30
    x[9, :500] = -1e30
    case["drafts"][:4] = torch.tensor([1, 2, 999, 17], dtype=torch.int32)
    case["drafts"][4:8] = torch.tensor([0, 3, 5, 4], dtype=torch.int32)
    case["uniforms"][:8] = 0.0
    check(case)


def test_drafts_outside_the_vocabulary_and_certain_ones():
    case = make([3, 2, 2, 2], 300, [PLAIN, (0.0, 1.0, 0), (0.9, 0.9, 10), PLAIN], False, seed=4)
    case["drafts"][:] = torch.tensor([-1, 0, 0, 300, 1, 2 ** 31 - 1, 0, 5, 6], dtype=torch.int32)
    case["uniforms"][7:] = torch.tensor([0.0, 1.0 - 2.0 ** -24], device="cuda")
    check(case)


def test_the_draft_is_the_target():
    """q equal to p but for rounding: nearly every draft passes, and where one does not the next token is still one of the target's."""
    case = make([6] * 20, 2000, [(1.0, 1.0, 0)], True, seed=5)
    starts = case["draft_start"].tolist()
    rows = [starts[r] + r + i for r in range(20) for i in range(6)]
    case["draft_probs"] = torch.softmax(case["logits"][rows].double(), -1).float()
    case["drafts"] = (case["draft_probs"] / torch.empty_like(case["draft_probs"]).exponential_(generator=torch.Generator(device="cuda").manual_seed(1))).argmax(-1).int()
    case["uniforms"].clamp_(max=0.999)
    accepted, token, _ = verify(case)
    assert accepted.tolist() == [6] * 20
    case["draft_probs"] = torch.ones_like(case["draft_probs"])           # covers the target everywhere: what is left is the target itself
    case["uniforms"].fill_(0.9999999)
    check(case)


@pytest.mark.parametrize("setting,vocab", [((0.9, 1.0, 0), 8), ((1.2, 0.8, 6), 12)])
@pytest.mark.parametrize("probabilities", [True, False])
def test_tokens_are_distributed_as_the_target(setting, vocab, probabilities):
    """The first token behind a prompt, drafted or not, has the target's distribution: 30,000 requests with one draft each, drawn from the draft's
    distribution.  A share of n draws has a standard deviation of at most 0.5 / sqrt(n): six of them are 0.0174."""
    n = 30000
    g = torch.Generator(device="cuda").manual_seed(11)
    row = 1.5 * torch.randn(vocab, generator=g, device="cuda")
    q = torch.softmax(torch.randn(vocab, generator=g, device="cuda"), -1)
    p = distribution(row, setting)
    if probabilities:
        drafts = torch.multinomial(q, n, replacement=True, generator=g).int()
    else:
        drafts = torch.full((n,), int(q.argmax()), dtype=torch.int32, device="cuda")
    case = dict(logits=row.expand(2 * n, vocab).contiguous(), drafts=drafts, draft_start=torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                uniforms=torch.rand(n, generator=g, device="cuda"), noise=torch.empty(n, vocab, device="cuda").exponential_(generator=g),
                draft_probs=q.expand(n, vocab).contiguous() if probabilities else None, records=records_of([setting]),
                slot_of_request=torch.zeros(n, dtype=torch.int32, device="cuda"))
    accepted, token, _ = verify(case)
    first = torch.where(accepted > 0, drafts, token).long()
    share = torch.bincount(first, minlength=vocab).double() / n
    assert float((share - p).abs().max()) < 6 * 0.5 / n ** 0.5
    kept = accepted.float().mean().item()
    rule = float(torch.minimum(p, q.double()).sum()) if probabilities else float(p[int(q.argmax())])
    assert abs(kept - rule) < 6 * 0.5 / n ** 0.5


def test_without_records_every_row_is_argmax():
    case = make([3, 0, 2], 700, [GREEDY], False, seed=6)
    accepted, token = (torch.empty(3, dtype=torch.int32, device="cuda") for _ in range(2))
    kernels.verify_drafts(case["logits"], case["drafts"], case["draft_start"], None, None, accepted, token)
    want = expected(case)
    assert accepted.tolist() == want[0] and token.tolist() == want[1]
    # greedy drafts give what sampling one by one gives: the argmax of every row
    best = torch.empty(8, dtype=torch.int32, device="cuda")
    kernels.sample(case["logits"], None, None, None, best)
    starts = [0, 4, 5]
    for r, start in enumerate(starts):
        assert token[r] == best[start + int(accepted[r])]


def test_no_drafts_is_a_draw_from_every_row():
    check(make([0, 0, 0, 0], 5000, [PLAIN, GREEDY, (1.0, 0.7, 50)], False, seed=7))


def test_captured_and_on_another_stream():
    first, second = (make([3, 1, 4], 3001, [PLAIN, (0.7, 0.9, 30), GREEDY], True, seed=s) for s in (8, 9))
    held = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in first.items()}
    verify(held)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = verify(held)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for case in (second, first):
            for k, v in case.items():
                if isinstance(v, torch.Tensor):
                    held[k].copy_(v)
            graph.replay()
            stream.synchronize()
            want = expected(case)
            assert out[0].tolist() == want[0] and out[1].tolist() == want[1]


def test_refusals():
    case = make([2, 1], 100, [PLAIN], True, seed=1)
    total, count = 3, 2
    ok = dict(logits=case["logits"], drafts=case["drafts"], draft_start=case["draft_start"], uniforms=case["uniforms"], noise=case["noise"],
              accepted=torch.zeros(count, dtype=torch.int32, device="cuda"), next_token=torch.zeros(count, dtype=torch.int32, device="cuda"),
              draft_probs=case["draft_probs"], records=case["records"], slot_of_request=case["slot_of_request"], target_probs=torch.zeros(total, device="cuda"))
    for other in (dict(logits=case["logits"].cpu()), dict(logits=case["logits"].bfloat16()), dict(logits=case["logits"][:4]), dict(logits=case["logits"][0]),
                  dict(logits=case["logits"].t()), dict(drafts=case["drafts"].long()), dict(draft_start=case["draft_start"][:2]), dict(uniforms=None),
                  dict(noise=None), dict(noise=case["noise"][:1]), dict(noise=case["noise"][:, :99]), dict(uniforms=case["uniforms"].double()),
                  dict(draft_probs=case["draft_probs"][:2]), dict(records=case["records"][:, :7]), dict(records=case["records"].float()),
                  dict(slot_of_request=None), dict(slot_of_request=case["slot_of_request"].long()), dict(next_token=torch.zeros(3, dtype=torch.int32, device="cuda")),
                  dict(accepted=torch.zeros(2, device="cuda")), dict(target_probs=torch.zeros(2, device="cuda"))):
        with pytest.raises(KernelError):
            kernels.verify_drafts(**{**ok, **other})
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    kernels.verify_drafts(torch.zeros((0, 100), device="cuda"), empty, torch.zeros(1, dtype=torch.int32, device="cuda"), None, None, empty, empty.clone())


def _numbers_on_borders(temperature, borders, most):
    """Distances from the largest logit that float32 products round onto a border, in eighths of a temperature, while the exact product lies beside it."""
    eighths = torch.tensor(8.0) / torch.tensor(temperature)
    found = []
    for border in torch.tensor(borders):
        distance = border / eighths
        for steps in range(-3, 4):
            d = (distance.view(torch.int32) + steps).view(torch.float32)
            if d * eighths == border and d.double() * eighths.double() != border.double():
                found.append(float(d))
    return found[::max(1, len(found) // most)][:most]


@pytest.mark.parametrize("vocab", [1200, 40000])
@pytest.mark.parametrize("temperature", [1.3, 0.8])
@pytest.mark.parametrize("borders", [[40.5 + part / 256.0 for part in range(1, 256)], [part + 0.5 for part in range(12, 120)]], ids=["parts", "bins"])
def test_masses_of_numbers_on_a_border(borders, temperature, vocab):
    """300 equal logits in whose middle the nucleus ends, where a rounding decides which of two neighbouring bins, or parts of one, holds them; some larger and some
    smaller ones beside them in either."""
    settings, rows, first = [], [], []
    g = torch.Generator().manual_seed(2)
    for distance in _numbers_on_borders(temperature, borders, 40):
        near = 0.4 / 256.0 * temperature / 8.0
        x = torch.full((vocab,), -float("inf"))
        places = torch.randperm(vocab, generator=g)[:451]
        x[places[0]] = 0.0
        x[places[1:51]], x[places[51:351]], x[places[351:]] = near - distance, -distance, -distance - near
        mass = torch.exp(x.double() / struct.unpack("f", struct.pack("f", temperature))[0])
        settings.append((temperature, float((mass[places[:51]].sum() + 150.5 * mass[places[51]]) / mass.sum()), 0))
        rows.append(x)
        first.append(int(places[51:351].min()))
    count = len(rows)
    assert count > 20
    logits = torch.stack(rows).repeat_interleave(2, 0).cuda()
    case = dict(logits=logits, drafts=torch.tensor(first, dtype=torch.int32).cuda(), draft_start=torch.arange(count + 1, dtype=torch.int32).cuda(),
                uniforms=torch.full((count,), 0.9, device="cuda"), noise=torch.empty(count, vocab, device="cuda").exponential_(generator=torch.Generator("cuda").manual_seed(3)),
                draft_probs=None, records=records_of(settings), slot_of_request=torch.arange(count, dtype=torch.int32).cuda(), settings=settings)
    check(case)


@pytest.mark.parametrize("settings", [[(1.0, 0.9, 0), (1.3, 0.5, 0)], [(1.0, 1.0, 20000), (0.8, 0.95, 30000)]])
def test_flat_rows(settings):
    """Logits that lie close together, so that an eighth of a temperature at the border holds thousands of a block's entries: few large blocks (more rows than have
    two each) and some of equal numbers."""
    check(make([1] * 205, 64000, settings, True, seed=12, spread=0.5))
    check(make([1] * 205, 40000, settings, False, seed=13, spread=0.3, grid=2.0 ** -10))


def test_flat_rows_take_no_other_way():
    """Flat rows are searched as peaked ones are: of 408 rows, which have a block each, they may take several times as long (their search reads them again and counts
    thousands of entries), not the twenty times that rounds over the bits of all numbers took."""
    def time_of(spread):
        case = make([3] * 102, 151936, [(1.0, 0.95, 0)], False, seed=14, spread=spread)
        for _ in range(3):
            verify(case)
        times = []
        for _ in range(5):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            verify(case)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        return sorted(times)[2]

    peaked, flat = time_of(3.0), time_of(1.0)
    assert flat < 9.0 * peaked, f"{flat:.3f} ms, {peaked:.3f} ms where few entries hold the mass"

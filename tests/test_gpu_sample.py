"""Sampling against its definition in 64 bits (run with -m gpu).

Tokens are equal. Weights are good to 2e-13 of themselves, sums of up to 2^18 of
them as well, so a decision that was made by more than 1e-9 of the sums compared
cannot fall otherwise; the cases' inputs are drawn so that every one is (checked:
room), or are exact by construction (equal logits). Shares are rounded to f32 once:
2^-24 of them, and 1e-12.
"""
import math

import numpy as np
import pytest

from sample_model import sample

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from kestrel_b200.cuda import Context
    c = Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def floats(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def run(ctx, logits, u, **settings):
    """(tokens, shares); settings: a value for all rows, or one for each."""
    n = logits.shape[0]
    row = lambda x, t: None if x is None else torch.tensor(list(x) if np.ndim(x) else [x] * n, dtype=t, device="cuda")
    tokens = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    probs = torch.full((n,), -7.0, device="cuda")
    ctx.sample_dev(logits, floats(u), tokens, probs=probs, temperature=row(settings.get("temperature"), F32),
                   top_k=row(settings.get("top_k"), torch.int32), top_p=row(settings.get("top_p"), F32),
                   min_p=row(settings.get("min_p"), F32))
    ctx.sync()
    return tokens.tolist(), probs.tolist()


def check(ctx, logits, u, sure=True, **settings):
    tokens, probs = run(ctx, logits, u, **settings)
    wide = logits.float().cpu().numpy()
    skipped = 0
    for i, (t, p) in enumerate(zip(tokens, probs)):
        one = {k: float(np.float32(np.asarray(v).reshape(-1)[i if np.ndim(v) else 0])) if k != "top_k" else
               int(np.asarray(v).reshape(-1)[i if np.ndim(v) else 0]) for k, v in settings.items()}
        want, share, room = sample(wide[i], float(np.float32(u[i])), **one)
        if sure and room < 1e-9:
            skipped += 1
            continue
        assert t == want, (i, t, want, one, u[i], room)
        assert abs(p - share) <= 2.0 ** -24 * share + 1e-12, (i, p, share)
    assert skipped <= len(tokens) // 20  # (a border of 1e-9 is rare)
    return tokens


def logits_of(n, vocab, t, seed, spread=2.2, lead=12.0):
    rng = np.random.default_rng(seed)
    x = spread * rng.standard_normal((n, vocab))
    for i in range(n):
        who = rng.integers(0, vocab, min(vocab, 30))
        x[i, who] += lead * rng.random() * rng.random(len(who))
    return torch.tensor(x, dtype=F32, device="cuda").to(t)


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=40), dict(top_k=1), dict(top_p=0.9), dict(top_p=0.05),
            dict(min_p=0.1), dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.02), dict(temperature=0.0),
            dict(temperature=1.5, top_k=700, top_p=0.99), dict(temperature=0.3, top_p=0.999, min_p=1e-6),
            dict(temperature=5.0, top_p=0.5), dict(top_k=2000, top_p=0.7), dict(min_p=1.0), dict(min_p=3.0)]


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_sample(ctx, settings, t):
    """Vocabularies from two tokens to several blocks' worth, odd ones among them."""
    for n, vocab in ((1, 2), (3, 7), (5, 1000), (2, 4096), (4, 32001), (2, 50257)):
        rng = np.random.default_rng(vocab)
        check(ctx, logits_of(n, vocab, t, vocab + n), rng.random(n).astype(np.float32), **settings)


@pytest.mark.parametrize("t", [F32, BF16], ids=str)
def test_many_rows_each_its_own(ctx, t):
    """A settings array per row, every block shape: few and many rows."""
    for n, vocab in ((1, 151936), (7, 151936), (40, 30000), (300, 501)):
        rng = np.random.default_rng(n)
        pick = lambda v: [v[i] for i in rng.integers(0, len(v), n)]
        check(ctx, logits_of(n, vocab, t, n), rng.random(n).astype(np.float32), temperature=pick([0.0, 0.5, 1.0, 1.3]),
              top_k=pick([0, -3, 1, 5, 100, 1000, vocab, vocab + 9]), top_p=pick([0.3, 0.9, 0.97, 1.0, 2.0]),
              min_p=pick([0.0, -1.0, 0.05]))


def test_the_largest_vocabulary(ctx):
    check(ctx, logits_of(2, 393216, F32, 1), [0.3, 0.8], top_p=0.9)
    check(ctx, logits_of(2, 393216, F16, 2), [0.3, 0.8], temperature=0.9, top_k=300)


def test_equal_logits(ctx):
    """Ties everywhere: cuts fall by index, borders at whole shares are exact;
    more equal tokens than one block looks through."""
    for n_vocab in (8, 4096, 65536):
        x = torch.full((6, n_vocab), -3.25, device="cuda")
        tokens, probs = run(ctx, x, [0.0, 0.25, 0.5, 0.75, 0.999999, 0.5])
        assert tokens == [0, n_vocab // 4, n_vocab // 2, 3 * n_vocab // 4, math.floor(n_vocab * float(np.float32(0.999999))), n_vocab // 2]
        assert probs == [1 / n_vocab] * 6
        tokens, probs = run(ctx, x, [0.0, 0.5, 0.99999, 0.5, 0.5, 0.5], top_p=0.5)
        assert tokens[:3] == [0, n_vocab // 4, n_vocab // 2 - 1] and probs[0] == 2 / n_vocab
        k = n_vocab // 2 + 1
        tokens, _ = run(ctx, x, [0.999999] * 6, top_k=k)
        assert tokens == [math.floor(k * float(np.float32(0.999999)))] * 6
        tokens, _ = run(ctx, x, [0.999999] * 6, top_k=k, top_p=0.5)
        need = math.ceil(k / 2)
        assert tokens == [math.floor(need * float(np.float32(0.999999)))] * 6
    # Two values, the border among the lower ones.
    x = torch.zeros((1, 40000), device="cuda")
    x[0, 1::2] = 1.0
    assert run(ctx, x, [0.9999999], top_k=20003)[0] == [39999]
    assert run(ctx, x, [0.0], top_k=20003)[0] == [0]
    assert run(ctx, x, [1e-5], top_k=20003, temperature=1e9)[0] == [0]


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=str)
def test_odd_logits(ctx, t):
    inf, nan = float("inf"), float("nan")
    for vocab in (5, 3000, 40000):
        x = torch.full((10, vocab), -inf, device="cuda", dtype=t)
        x[1, 3] = -5.0                       # one token
        x[2, :] = nan                        # nothing
        x[3, 2], x[3, 4] = inf, inf          # infinite ones share
        x[4, :] = torch.finfo(t).min         # the type's lowest, all
        x[5, :] = torch.finfo(t).min
        x[5, 1] = 0.0
        x[6, 0], x[6, 4] = nan, 2.0
        x[7, 0], x[7, 1], x[7, 2] = -0.0, 0.0, -0.0  # zeros are equal
        x[8, 1], x[8, 3] = 1.0, 1.0
        x[9, :] = torch.finfo(t).max
        for settings in (dict(), dict(top_k=2), dict(top_p=0.5), dict(top_k=3, top_p=0.9, min_p=0.1), dict(temperature=0.0),
                         dict(temperature=float("inf")), dict(temperature=1e-30), dict(temperature=nan)):
            u = [0.6] * 10
            tokens = check(ctx, x, u, sure=False, **settings)
            assert tokens[0] == tokens[2] == -1 and tokens[1] == 3 and tokens[6] == 4


def test_settings_and_numbers_out_of_range(ctx):
    x = logits_of(4, 2000, F32, 5)
    for u in ([-1.0, float("nan"), 0.0, -0.0], [1.0, 2.0, float("inf"), 1 - 2.0 ** -24]):
        for settings in (dict(), dict(top_k=10), dict(top_p=0.6)):
            check(ctx, x, u, sure=False, **settings)
    nan = float("nan")
    same = run(ctx, x, [0.1, 0.4, 0.7, 0.9])
    assert run(ctx, x, [0.1, 0.4, 0.7, 0.9], top_p=nan, min_p=nan, top_k=0, temperature=1.0) == same
    assert run(ctx, x, [0.5] * 4, top_p=-1.0) == run(ctx, x, [0.5] * 4, top_p=0.0) == run(ctx, x, [0.5] * 4, top_k=1)


def test_rows_of_any_stride_and_place(ctx):
    """Rows that are slices of wider ones, at odd offsets; probs not wanted."""
    for t in (F32, F16):
        for pad, vocab in ((1, 3001), (4, 5000), (0, 777)):
            buf = logits_of(5, vocab + 2 * pad + 3, t, pad)
            x = buf[:, pad:pad + vocab]
            want = check(ctx, x, [0.05, 0.3, 0.5, 0.7, 0.95], temperature=0.9, top_p=0.95)
            tokens = torch.empty(5, dtype=torch.int32, device="cuda")
            ctx.sample_dev(x, floats([0.05, 0.3, 0.5, 0.7, 0.95]), tokens, temperature=floats([0.9] * 5),
                           top_p=floats([0.95] * 5))
            ctx.sync()
            assert tokens.tolist() == want


def test_peaks_and_gaps(ctx):
    """Rows whose sums lie in a few tokens, with empty bins between, and rows whose
    bins at the border hold thousands."""
    rng = np.random.default_rng(0)
    rows = []
    for gap in (0.5, 3.0, 11.0, 23.5, 30.0):
        x = -gap + 0.001 * rng.standard_normal(30000)
        x[[17, 29999]] = 0.0, -0.1
        rows.append(x)
    rows.append(1e-4 * rng.standard_normal(30000))
    rows.append(np.linspace(0, -200, 30000))
    rows.append(np.linspace(-1, 1, 30000) ** 9 * 40)
    x = torch.tensor(np.array(rows), dtype=F32, device="cuda")
    for settings in (dict(), dict(top_p=0.9), dict(top_p=0.5), dict(top_p=0.9999), dict(top_k=100), dict(top_k=9000),
                     dict(top_k=9000, top_p=0.8), dict(temperature=0.05, top_p=0.9), dict(temperature=40.0, top_p=0.9),
                     dict(temperature=0.05, top_k=15000, top_p=0.99)):
        for u in (0.02, 0.5, 0.97):
            check(ctx, x, [u] * len(rows), sure=True, **settings)


def test_draws_follow_the_shares(ctx):
    """Over evenly spaced numbers every token comes up as often as its share says,
    but for one at each border."""
    l = torch.tensor([[0.3, -1.0, 2.0, 0.0, 1.1, -4.0]], device="cuda")
    n = 4096
    tokens, probs = run(ctx, l.expand(n, 6), (np.arange(n) + 0.5) / n, temperature=0.9, min_p=0.03)
    w = np.exp((l.cpu().double().numpy()[0] - 2.0) / np.float32(0.9))
    w[w < 0.03] = 0
    for j in range(6):
        assert abs(tokens.count(j) - n * w[j] / w.sum()) <= 1.0
    for t, p in zip(tokens, probs):
        assert abs(p - w[t] / w.sum()) < 1e-7


def test_repeats_and_graphs(ctx):
    """The same bits every time; captured, and replayed with other numbers."""
    x = logits_of(64, 20000, F32, 3)
    u = np.random.default_rng(1).random(64).astype(np.float32)
    settings = dict(temperature=1.1, top_k=3000, top_p=0.9)
    first = run(ctx, x, u, **settings)
    for _ in range(3):
        assert run(ctx, x, u, **settings) == first
    tokens, u_dev = torch.zeros(64, dtype=torch.int32, device="cuda"), floats([0.5] * 64)
    args = dict(temperature=floats([1.1] * 64), top_k=torch.full((64,), 3000, dtype=torch.int32, device="cuda"),
                top_p=floats([0.9] * 64))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(stream.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ctx.sample_dev(x, u_dev, tokens, **args)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    u_dev.copy_(floats(u))
    graph.replay()
    torch.cuda.synchronize()
    assert tokens.tolist() == first[0]


def test_refusals(ctx):
    from kestrel_b200.cuda import KestrelCudaError
    x, u, tokens = torch.zeros((2, 8), device="cuda"), floats([0.5, 0.5]), torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(KestrelCudaError) as e:
        ctx.sample_dev(torch.zeros((1, 393217), device="cuda"), u[:1], tokens[:1])
    assert e.value.code == 2
    with pytest.raises(KestrelCudaError) as e:
        ctx.sample_dev(x[:, :0], u, tokens)
    assert e.value.code == 2
    for bad in (lambda: ctx.sample_dev(x, None, tokens), lambda: ctx.sample_dev(x, u[:1], tokens),
                lambda: ctx.sample_dev(x, u, tokens.float()), lambda: ctx.sample_dev(x.double(), u, tokens),
                lambda: ctx.sample_dev(x.t(), u, tokens), lambda: ctx.sample_dev(x, u, tokens, top_k=u),
                lambda: ctx.sample_dev(x, u, tokens, top_p=u.cpu()), lambda: ctx.sample_dev(x, u, tokens, probs=u[:1])):
        with pytest.raises(ValueError):
            bad()
    ctx.sample_dev(x[:0], u[:0], tokens[:0])
    ctx.sync()

"""control_logits and sample_each (serving/controls.py) against the 64-bit restatement
oracle/requests_ref.py.

Controls: half a step of the type on the result, and at most four fp32 operations, each
off by 2^-24 of what it has (the logit times or over the repetition, the penalties, the
biases). A draw is the oracle's id where u is further from the next border than the
weights' rounding: 2^-44 of the largest weight each, so vocab * 2^-44 of their sum."""
import numpy as np
import pytest
import torch

from oracle import requests_ref as ref
from serving import _native
from serving.controls import LogitControls, control_logits, sample_each

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def f32(x):
    return torch.tensor(np.asarray(x), dtype=torch.float32, device=DEV)


def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def pack(allowed):
    """bool [masks, vocab] -> int32 [masks, words]."""
    n, v = allowed.shape
    bits = np.zeros((n, -(-v // 32) * 32), dtype=np.uint8)
    bits[:, :v] = allowed
    return i32(np.packbits(bits, axis=1, bitorder="little").view(np.int32))


class Problem:
    def __init__(self, rows, vocab, cap, n_bias, n_masks, dtype, seed=0):
        rng = np.random.default_rng([rows, vocab, cap, n_bias, n_masks, seed])
        self.rows, self.vocab, self.dtype = rows, vocab, dtype
        self.logits = torch.from_numpy(rng.normal(0, 3, (rows, vocab))).to(dtype)
        # a few ids make up most of the history, so counts go past one
        self.tokens = np.where(rng.random((rows, cap)) < 0.6,
                               rng.integers(0, max(1, vocab // 20), (rows, cap)),
                               rng.integers(0, vocab, (rows, cap)))
        self.lens = rng.integers(0, cap + 1, rows)
        self.lens[rng.integers(0, rows)] = cap
        self.prompt = (self.lens * rng.random(rows)).astype(np.int64)
        self.repetition = rng.choice([1.0, 0.8, 1.1, 1.7], rows).astype(np.float32)
        self.presence = rng.choice([0.0, 0.5, -0.25], rows).astype(np.float32)
        self.frequency = rng.choice([0.0, 0.3, 0.1], rows).astype(np.float32)
        per = rng.integers(0, n_bias + 1, rows)
        self.starts = np.concatenate([[0], np.cumsum(per)])
        self.bias_ids = rng.integers(0, vocab, self.starts[-1])
        self.bias_values = rng.choice([-100.0, 0.1, 0.7, 3.3, 1e-3],
                                      self.starts[-1]).astype(np.float32)
        self.allowed = rng.random((n_masks, vocab)) < rng.random((n_masks, 1))
        self.mask_rows = rng.integers(-1, n_masks, rows) if n_masks else np.full(rows, -1)

    def controls(self, history=True, bias=True, mask=True):
        kw = {}
        if history:
            kw.update(tokens=i32(self.tokens), lens=i32(self.lens), prompt_lens=i32(self.prompt),
                      repetition=f32(self.repetition), presence=f32(self.presence),
                      frequency=f32(self.frequency))
        if bias:
            kw.update(bias_ids=i32(self.bias_ids), bias_values=f32(self.bias_values),
                      bias_starts=i32(self.starts))
        if mask:
            kw.update(masks=pack(self.allowed), mask_rows=i32(self.mask_rows))
        return LogitControls(**kw)

    def check(self, got, history=True, bias=True, mask=True):
        x = self.logits.double().numpy()
        got = got.cpu().double().numpy()
        for r in range(self.rows):
            biases = []
            if bias:
                a, b = self.starts[r], self.starts[r + 1]
                biases = [(int(t), float(v)) for t, v in zip(self.bias_ids[a:b],
                                                              self.bias_values[a:b])]
            toks = self.tokens[r, :self.lens[r]] if history else []
            allowed = self.allowed[self.mask_rows[r]] if mask and self.mask_rows[r] >= 0 else None
            pars = [float(p[r]) for p in (self.repetition, self.presence, self.frequency)]
            want = ref.control(x[r], toks, int(self.prompt[r]), *pars, biases, allowed)
            # every operation's operands and results are below the sum of the magnitudes
            size = np.abs(x[r]) * max(pars[0], 1 / pars[0]) + abs(pars[1]) + abs(pars[2]) * len(toks)
            for t, v in biases:
                size[t] += abs(v)
            ops = 4 + len(biases)
            tol = torch.finfo(self.dtype).eps / 2 * np.abs(want) + ops * 2.0 ** -24 * size
            gone = np.isinf(want)
            assert np.array_equal(np.isneginf(got[r]), gone)
            err = np.abs(got[r][~gone] - want[~gone])
            assert (err <= tol[~gone] * (1 + 2.0 ** -7)).all(), (r, float((err - tol[~gone]).max()))


SHAPES = [(1, 1, 3, 2, 1), (2, 7, 5, 3, 2), (3, 31, 0, 0, 1), (5, 33, 40, 9, 3),
          (40, 100, 300, 20, 4), (4, 50257, 500, 30, 2), (33, 4097, 1000, 700, 3),
          (64, 9001, 64, 5, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_control_logits(shape, dtype):
    print(f"[controls] {shape} {dtype}", flush=True)
    p = Problem(*shape, dtype)
    x = p.logits.to(DEV)
    for kinds in ((True, True, True), (True, False, False), (False, True, False),
                  (False, False, True)):
        kw = dict(zip(("history", "bias", "mask"), kinds))
        c = p.controls(**kw)
        st = status()
        out = control_logits(x, c, status=st)
        assert int(st) == 0
        p.check(out, **kw)
        assert torch.equal(x.cpu(), p.logits)
        # the same bits in place, and where rows start anywhere
        y = x.clone()
        assert control_logits(y, c, out=y) is y and torch.equal(y, out)
        wide = torch.zeros(p.rows, p.vocab + 5, dtype=dtype, device=DEV)
        src = torch.zeros(p.rows, p.vocab + 3, dtype=dtype, device=DEV)
        src[:, 1:1 + p.vocab] = x
        control_logits(src[:, 1:1 + p.vocab], c, out=wide[:, 2:2 + p.vocab])
        assert torch.equal(wide[:, 2:2 + p.vocab], out)
        assert not wide[:, :2].any() and not wide[:, 2 + p.vocab:].any()
    assert torch.equal(control_logits(x, LogitControls()), x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1100, 90, 20, 4, 2), (85, 50257, 300, 40, 2)])
def test_control_logits_of_many_workgroups(shape, dtype):
    print(f"[controls] {shape} {dtype}", flush=True)
    p = Problem(*shape, dtype)
    x = p.logits.to(DEV)
    p.check(control_logits(x, p.controls()))
    wide = torch.zeros(p.rows, p.vocab + 5, dtype=dtype, device=DEV)
    y = wide[:, 3:3 + p.vocab]
    y.copy_(x)
    p.check(control_logits(y, p.controls(), out=y))
    assert not wide[:, :3].any() and not wide[:, 3 + p.vocab:].any()


def test_biases_that_share_places():
    """Ids whose places collide, each of them several times, more than a batch of them."""
    rng = np.random.default_rng(12)
    vocab = 60000
    ids = rng.choice(np.arange(0, vocab, 1024), 1500)
    values = rng.choice([1.0, -3.0, 1e-3, 1e4], 1500).astype(np.float32)
    x = torch.zeros(1, vocab, device=DEV)
    c = LogitControls(bias_ids=i32(ids), bias_values=f32(values), bias_starts=i32([0, 1500]))
    want = np.zeros(vocab, dtype=np.float32)
    for i, v in zip(ids, values):
        want[i] = np.float32(want[i] + v)  # in the list's order, rounded at every step
    assert np.array_equal(control_logits(x, c)[0].cpu().numpy(), want)


def test_an_id_named_many_times_is_added_up_in_order():
    """Values whose sum depends on the order: 1e8, 1, -1e8, 1 in fp32 gives 1; and lists
    longer than a workgroup, of one id and of two in turn."""
    x = torch.zeros(1, 40, device=DEV)

    def sums(ids, values):
        c = LogitControls(bias_ids=i32(ids), bias_values=f32(values), bias_starts=i32([0, len(ids)]))
        return control_logits(x, c)[0].tolist()

    assert sums([5, 5, 5, 5], [1e8, 1.0, -1e8, 1.0])[5] == 1.0
    rng = np.random.default_rng(4)
    values = rng.normal(0, 1, 1300).astype(np.float32) * rng.choice([1, 1e6], 1300)
    for ids in ([7] * 1300, [3, 9] * 650):
        want = [np.float32(0)] * 40
        for t, v in zip(ids, values.astype(np.float32)):
            want[t] = np.float32(want[t] + v)
        assert sums(ids, values) == [float(w) for w in want]


def test_logits_that_are_not_finite():
    x = torch.tensor([[INF, -INF, float("nan"), 1.0, -1.0]], device=DEV)
    c = LogitControls(tokens=i32([[0, 1, 2, 3, 4]]), lens=i32([5]), repetition=f32([2.0]),
                      frequency=f32([0.5]), bias_ids=i32([1, 0]), bias_values=f32([INF, 1.0]),
                      bias_starts=i32([0, 2]))
    out = control_logits(x, c)[0].tolist()
    assert out[0] == INF and np.isnan(out[1]) and np.isnan(out[2]) and out[3:] == [0.0, -2.5]
    # a mask's -infinity takes the place of whatever was there
    c = LogitControls(masks=i32([[0b11000]]), mask_rows=i32([0]))
    assert control_logits(x, c)[0].tolist() == [-INF, -INF, -INF, 1.0, -1.0]
    c = LogitControls(masks=i32([[0]]), mask_rows=i32([0]))  # a mask that leaves nothing
    assert control_logits(x, c)[0].tolist() == [-INF] * 5


def test_what_is_out_of_range_is_skipped_and_reported():
    x = torch.arange(1.0, 9.0, device=DEV)[None].repeat(3, 1)

    def run(**kw):
        st = status()
        return control_logits(x, LogitControls(**kw), status=st), int(st)

    tok = i32([[1, -1, 8, 2], [3, 3, 3, 3], [2 ** 31 - 1, 0, 0, 0]])
    out, bits = run(tokens=tok, lens=i32([4, 0, 1]), presence=f32([1.0, 1.0, 1.0]))
    want = x.clone()
    want[0, 1] -= 1
    want[0, 2] -= 1
    assert bits == _native.PKV_STATUS_BAD_TOKEN and torch.equal(out, want)
    # lengths past the tensor are cut, negative ones are none
    out, bits = run(tokens=i32([[1], [2], [3]]), lens=i32([9, -1, 1]), prompt_lens=i32([0, 0, 2]),
                    presence=f32([1.0, 1.0, 1.0]))
    want = x.clone()
    want[0, 1] -= 1
    assert bits == _native.PKV_STATUS_BAD_CONTROL and torch.equal(out, want)
    out, bits = run(bias_ids=i32([0, 8, -1]), bias_values=f32([1, 1, 1]), bias_starts=i32([0, 3, 3, 9]))
    want = x.clone()
    want[0, 0] += 1
    assert bits == _native.PKV_STATUS_BAD_TOKEN | _native.PKV_STATUS_BAD_CONTROL
    assert torch.equal(out, want)
    out, bits = run(masks=i32([[0]]), mask_rows=i32([1, -2, -1]))
    assert bits == _native.PKV_STATUS_BAD_CONTROL and torch.equal(out, x)


def test_control_refusals():
    x = torch.zeros(2, 64, device=DEV)
    one = i32([0, 0])
    with pytest.raises(ValueError, match="go together"):
        LogitControls(tokens=i32([[1], [2]]))
    with pytest.raises(ValueError, match="go together"):
        LogitControls(masks=i32([[0, 0]]))
    with pytest.raises(ValueError, match="needs tokens"):
        LogitControls(presence=f32([0, 0]))
    with pytest.raises(ValueError, match="disagree"):
        LogitControls(tokens=i32([[1], [2]]), lens=one, masks=i32([[0, 0]]), mask_rows=i32([0]))
    with pytest.raises(ValueError, match="lens"):
        LogitControls(tokens=i32([[1], [2]]), lens=one.long())
    with pytest.raises(ValueError, match="share a device"):
        LogitControls(tokens=i32([[1], [2]]), lens=one.cpu())
    with pytest.raises(ValueError, match="controls of 1 rows"):
        control_logits(x, LogitControls(masks=i32([[0, 0]]), mask_rows=i32([0])))
    with pytest.raises(ValueError, match="words"):
        control_logits(x, LogitControls(masks=i32([[0]]), mask_rows=one))
    with pytest.raises(ValueError, match="out must be"):
        control_logits(x, LogitControls(), out=x[:, :63])
    buf = torch.zeros(3, 64, device=DEV)
    with pytest.raises(ValueError, match="shares memory"):
        control_logits(buf[:2], LogitControls(), out=buf[1:])
    with pytest.raises(TypeError):
        control_logits(x.double(), LogitControls())
    with pytest.raises(RuntimeError):
        control_logits(x.cpu(), LogitControls())
    with pytest.raises(NotImplementedError):
        control_logits(x.clone().requires_grad_(), LogitControls())
    assert control_logits(x[:0], LogitControls()).shape == (0, 64)
    assert control_logits(x[:, :0], LogitControls()).shape == (2, 0)


# ---- draws -----------------------------------------------------------------

def draw_and_check(logits, temperature, top_k, top_p, min_p, u, least_checked=0.9):
    """logits [rows, vocab] on the device; parameters as lists, one a row."""
    rows, vocab = logits.shape
    st = status()
    ids, lp = sample_each(logits, f32(temperature), i32(top_k), f32(top_p), f32(min_p), f32(u),
                          status=st)
    assert int(st) == 0
    x = logits.double().cpu().numpy()
    ids, lp = ids.tolist(), lp.tolist()
    checked = 0
    for r in range(rows):
        want, logp, margin = ref.draw(x[r], *(float(np.float32(v)) for v in (temperature[r],)),
                                      int(top_k[r]), float(np.float32(top_p[r])),
                                      float(np.float32(min_p[r])), float(np.float32(u[r])))
        if margin < vocab * 2.0 ** -44 + 1e-12:
            continue
        checked += 1
        assert ids[r] == want, (r, temperature[r], top_k[r], top_p[r], min_p[r], u[r])
        # fp32's step on the result, and on its two parts the 64-bit steps
        assert abs(lp[r] - logp) <= 2.0 ** -23 * abs(logp) + vocab * 2.0 ** -42
    assert checked >= least_checked * rows


def params(rng, rows):
    return (rng.choice([0.0, 0.2, 0.7, 1.0, 1.9], rows), rng.choice([0, 1, 2, 30, 64, 65, 1000], rows),
            rng.choice([1.0, 0.99, 0.9, 0.5, 0.01], rows), rng.choice([0.0, 0.0, 0.05, 0.9, 1.0], rows),
            rng.random(rows, dtype=np.float32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,std", [(40, 1, 1), (40, 2, 1), (60, 37, 2), (90, 1000, 3),
                                            (60, 4099, 2.5), (60, 32001, 0.5), (24, 50257, 3),
                                            (6, 131072, 6)])
def test_sample_each(rows, vocab, std, dtype):
    print(f"[sample] {rows} {vocab} {dtype}", flush=True)
    rng = np.random.default_rng([rows, vocab])
    x = torch.from_numpy(rng.normal(0, std, (rows, vocab))).to(dtype).to(DEV)
    draw_and_check(x, *params(rng, rows))
    # rows that start anywhere, some ids masked
    wide = torch.zeros(rows, vocab + 9, dtype=dtype, device=DEV)
    y = wide[:, 3:3 + vocab]
    y.copy_(x)
    if vocab > 2:
        y[:, 1::2] = -INF
        y[::3, 4:] = -INF
    draw_and_check(y, *params(rng, rows))


@pytest.mark.parametrize("dtype", TYPES)
def test_ties(dtype):
    """All alike, two values, and the border of top-k and top-p inside a run of ties."""
    rng = np.random.default_rng(8)
    rows = 64
    for x in (np.zeros((rows, 3000)), rng.choice([1.0, 2.0], (rows, 3000)),
              rng.choice([-3.0, 0.0, 0.5, 4.0], (rows, 777)), np.full((rows, 5), -7.0),
              rng.integers(-3, 4, (rows, 20011)).astype(float)):
        t = torch.from_numpy(x).to(dtype).to(DEV)
        draw_and_check(t, *params(rng, rows), least_checked=0.6)
    zeros = torch.tensor([[0.0, -0.0, 0.0, -1.0]], device=DEV).to(dtype)  # -0 is 0
    ids = [int(sample_each(zeros, f32([1.0]), i32([2]), f32([1.0]), f32([0.0]), f32([u]))[0])
           for u in (0.0, 0.4, 0.7, 0.99)]
    assert ids == [0, 1, 2, 2]
    ids = [int(sample_each(zeros, f32([1.0]), None, f32([0.4]), None, f32([u]))[0])
           for u in (0.0, 0.49, 0.51, 0.99)]
    assert ids == [0, 0, 1, 1]  # weights 1 1 1 0.37: before the third it is 0.59 of the sum


@pytest.mark.parametrize("dtype", TYPES)
def test_more_values_than_are_listed(dtype):
    """Wide nuclei and large top_k, with few values near the border and with many; and borders
    further from the largest logit than the bins of the counts reach."""
    rng = np.random.default_rng(21)
    rows, vocab = 20, 50257
    u = rng.random(rows, dtype=np.float32)
    t = [1.0, 1.4, 0.7, 3.0] * 5
    k = [0] * 8 + [9000, 20000, 50256, 50257, 12000, 30000] * 2
    p = [0.95, 0.9, 0.999, 0.99] * 4 + [1.0] * 4
    m = [0.0, 0.0, 1e-3, 1e-6, 0.0] * 4
    for x in (rng.normal(0, 2, (rows, vocab)), rng.integers(-6, 7, (rows, vocab)) / 2.0,
              np.sort(rng.normal(0, 2, (rows, vocab)), axis=1)):
        draw_and_check(torch.from_numpy(x).to(dtype).to(DEV), t, k, p, m, u, least_checked=0.6)
    x = torch.from_numpy(rng.normal(0, 2, (rows, vocab))).to(dtype).to(DEV)
    draw_and_check(x, [0.01, 0.05, 0.2, 0.3] * 5, [40000, 1000, 300, 50000] * 5, p, m, u)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["mixed", "sorted", "ties"])
def test_a_row_draws_the_same_in_any_batch(dtype, order):
    """Few long rows are split over workgroups, many are not."""
    rng = np.random.default_rng(77)
    rows, vocab, times = 24, 50257, 26
    x = rng.normal(0, 2.5, (rows, vocab))
    if order == "sorted":  # what is kept lies together
        x = np.sort(x, axis=1)
    elif order == "ties":
        x = np.round(x)
    x = torch.from_numpy(x).to(dtype).to(DEV)
    t = [1.0, 0.7, 1.4, 0.0, 0.3, 3.0] * 4
    k = [0, 0, 0, 5, 400, 20000] * 2 + [0, 50, 0, 0, 0, 9000] * 2
    p = [1.0, 0.9, 0.95, 0.5] * 6
    m = [0.0, 0.0, 0.02, 0.0, 0.0, 0.1] * 4
    u = rng.random(rows, dtype=np.float32)
    few = sample_each(x, f32(t), i32(k), f32(p), f32(m), f32(u))
    many = sample_each(x.repeat(times, 1), f32(t * times), i32(k * times), f32(p * times),
                       f32(m * times), f32(u).repeat(times))
    assert torch.equal(few[0].repeat(times), many[0])
    assert torch.equal(few[1].repeat(times), many[1])
    for i in range(rows):  # and alone
        one = sample_each(x[i:i + 1], f32(t[i:i + 1]), i32(k[i:i + 1]), f32(p[i:i + 1]),
                          f32(m[i:i + 1]), f32(u[i:i + 1]))
        assert torch.equal(one[0], few[0][i:i + 1]) and torch.equal(one[1], few[1][i:i + 1])


def test_far_apart_and_extreme_parameters():
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.normal(0, 1, (32, 500)) * 1e4).float().to(DEV)
    x[:, 7] = 3e38
    x[1, 9] = -3e38
    x[2] = 0.0
    for temp in (1e-30, 1e-3, 1.0, 1e30, 3e38):
        n = len(x)
        draw_and_check(x, [temp] * n, [0, 3, 499, 500, 501, 2 ** 30] * 5 + [0, 1],
                       [1.0, 0.3, 1e-30, 1.5] * 8, [0.0, 1e-30, 0.5, 1.0] * 8,
                       rng.random(n, dtype=np.float32), least_checked=0.7)
    for u in (0.0, 1 - 2.0 ** -24):  # the ends of the uniforms
        draw_and_check(x, [0.7] * 32, [0] * 32, [0.9] * 32, [0.0] * 32, [u] * 32, least_checked=0)


def test_left_out_parameters_are_off():
    rng = np.random.default_rng(6)
    x = torch.from_numpy(rng.normal(0, 2, (20, 900))).float().to(DEV)
    t, u = f32(rng.choice([0.0, 0.8], 20)), f32(rng.random(20))
    a = sample_each(x, t, uniforms=u)
    b = sample_each(x, t, i32([0] * 20), f32([1.0] * 20), f32([0.0] * 20), u)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    torch.manual_seed(3)
    c = sample_each(x, t)
    torch.manual_seed(3)
    d = sample_each(x, t, uniforms=torch.rand(20, device=DEV))
    assert torch.equal(c[0], d[0])


def test_rows_that_cannot_be_drawn():
    x = torch.randn(9, 300, device=DEV)
    x[1, 299], x[2, 0], x[3], x[4, 1:] = float("nan"), INF, -INF, -INF
    n = len(x)
    temp, k, p, m, u = [1.0] * n, [0] * n, [1.0] * n, [0.0] * n, [0.5] * n
    temp[5], k[6], p[7], m[8] = -1.0, -1, 0.0, 1.5
    st = status()
    ids, lp = sample_each(x, f32(temp), i32(k), f32(p), f32(m), f32(u), status=st)
    assert ids[1:4].tolist() == [-1] * 3 and ids[5:].tolist() == [-1] * 4
    assert bool(lp[1:4].isnan().all()) and bool(lp[5:].isnan().all())
    assert int(ids[0]) >= 0 and int(ids[4]) == 0 and float(lp[4]) == 0.0
    assert int(st) == (_native.PKV_STATUS_NONFINITE | _native.PKV_STATUS_BAD_DISTRIBUTION
                       | _native.PKV_STATUS_BAD_CONTROL)
    for bad in (float("nan"), INF):
        assert sample_each(x[:1], f32([bad]))[0].tolist() == [-1]
    for bad in (1.0, -0.1, float("nan")):
        assert sample_each(x[:1], f32([1.0]), uniforms=f32([bad]))[0].tolist() == [-1]
    # a greedy row of NaN, too
    assert sample_each(x[1:2], f32([0.0]))[0].tolist() == [-1]


def test_sample_refusals():
    x = torch.randn(3, 20, device=DEV)
    t = f32([1.0] * 3)
    with pytest.raises(ValueError, match="temperature"):
        sample_each(x, t[:2])
    with pytest.raises(ValueError, match="top_k"):
        sample_each(x, t, top_k=t)
    with pytest.raises(ValueError, match="uniforms"):
        sample_each(x, t, uniforms=t.cpu())
    with pytest.raises(ValueError, match="logits"):
        sample_each(x[0], t)
    with pytest.raises(ValueError, match="logits"):
        sample_each(x[:, :0], t)
    with pytest.raises(RuntimeError):
        sample_each(x.cpu(), t)
    with pytest.raises(NotImplementedError):
        sample_each(x.clone().requires_grad_(), t)
    with torch.no_grad():
        sample_each(x.clone().requires_grad_(), t)
    with pytest.raises(TypeError):
        sample_each(x.double(), t)
    ids, lp = sample_each(x[:0], t[:0])
    assert ids.shape == (0,) and lp.shape == (0,)
    # columns at a stride and rows of one memory are copied
    assert sample_each(x.t().contiguous().t(), f32([0.0] * 3))[0].tolist() == x.argmax(1).tolist()
    assert sample_each(x[:1].expand(3, 20), f32([0.0] * 3))[0].tolist() == [int(x[0].argmax())] * 3


def test_the_widest_rows():
    rng = np.random.default_rng(31)
    wide = torch.zeros(2, (1 << 20) + 3, device=DEV)
    x = wide[:, 3:]
    x.copy_(torch.from_numpy(rng.normal(0, 2, (2, 1 << 20))).float())
    for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (1000, 0.9, 0.0), (0, 1.0, 0.3)):
        draw_and_check(x, [1.0, 0.6], [k] * 2, [p] * 2, [m] * 2, rng.random(2, dtype=np.float32),
                       least_checked=0.5)
    with pytest.raises(ValueError, match="logits"):
        sample_each(wide, f32([1.0, 1.0]))


def test_rows_that_are_gigabytes_apart():
    rows, vocab, far = 4, 1009, 1 << 30  # the last row begins past 2^31 elements
    buf = torch.empty(rows - 1, far, dtype=torch.bfloat16, device=DEV)
    x = buf.view(-1).as_strided((rows, vocab), (far - 1000, 1))
    p = Problem(rows, vocab, 30, 5, 2, torch.bfloat16)
    x.copy_(p.logits)
    t, u = f32([0.0, 0.7, 1.0, 1.0]), f32([0.1, 0.9, 0.5, 0.2])
    want = sample_each(p.logits.to(DEV), t, i32([0, 5, 0, 9]), None, None, u)
    got = sample_each(x, t, i32([0, 5, 0, 9]), None, None, u)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    p.check(control_logits(x, p.controls()))
    p.check(control_logits(x, p.controls(), out=x))


def test_two_streams_at_once():
    p = Problem(40, 20011, 300, 20, 4, torch.bfloat16)
    q = Problem(24, 20011, 300, 20, 4, torch.bfloat16, seed=1)
    rng = np.random.default_rng(9)
    work = []
    for a in (p, q):
        t, k, tp, mp, u = params(rng, a.rows)
        work.append((a.logits.to(DEV), a.controls(), f32(t), i32(k), f32(tp), f32(mp), f32(u)))

    def step(x, c, *pars):
        y = control_logits(x, c)
        return (y,) + sample_each(y, *pars)

    want = [step(*a) for a in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*work[i]))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(a, b) for r in runs for a, b in zip(w[:2], r[:2]))
        assert all(torch.equal(w[2].nan_to_num(9), r[2].nan_to_num(9)) for r in runs)


def test_both_in_a_graph():
    """Histories, parameters and logits change between replays."""
    p = Problem(6, 5003, 50, 10, 3, torch.bfloat16)
    c, x = p.controls(), p.logits.to(DEV)
    t, k, u = f32([0.0, 0.5, 1, 1, 1, 1]), i32([0, 0, 5, 50, 0, 0]), f32([0.5] * 6)
    top_p = f32([1.0, 1, 1, 0.9, 0.5, 1])

    def step():
        y = control_logits(x, c)
        return (y,) + sample_each(y, t, k, top_p, None, u)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for r in range(4):
        q = Problem(6, 5003, 50, 10, 3, torch.bfloat16, seed=r)
        x.copy_(q.logits)
        c.tokens.copy_(i32(q.tokens))
        c.lens.copy_(i32(q.lens))
        c.prompt_lens.copy_(i32(q.prompt))
        u.copy_(torch.rand(6))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))

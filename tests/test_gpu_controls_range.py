"""control_logits and sample_each at the ends of their types' range and past the sizes of a
single round.

Tolerances are those of tests/test_gpu_controls.py: half a step of the type on the result
and 2^-24 of the sum of the magnitudes for each fp32 operation."""
import numpy as np
import pytest
import torch

from oracle import requests_ref as ref
from serving.controls import LogitControls, control_logits, sample_each

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def f32(x):
    return torch.tensor(np.asarray(x), dtype=torch.float32, device=DEV)


@pytest.mark.parametrize("dtype", TYPES)
def test_finite_logits_under_finite_controls_stay_finite(dtype):
    """Results past the type's largest value are that value: a row a request's controls
    carry out of range can still be drawn."""
    most = float(torch.finfo(dtype).max)
    values = [3.0, -3.0, 0.0, 2.0 ** 15, most, -most, 1.0, -2.0 ** -10]
    cases = [  # repetition, presence, frequency, bias of every id
        (1e-30, 0.0, 0.0, 0.0), (1e-38, 0.0, 0.0, 0.0), (3e38, 0.0, 0.0, 0.0),
        (1.0, -1e5, 0.0, 0.0), (1.0, -3e38, 0.0, 0.0), (1.0, 3e38, 0.0, 0.0),
        (1.0, 0.0, -3e38, 0.0), (1.0, 0.0, 3e38, 0.0),
        (1.0, 0.0, 0.0, 3e38), (1.0, 0.0, 0.0, -3e38), (1.0, 0.0, 0.0, 1e5)]
    rows, vocab = len(cases), len(values)
    x = torch.tensor(values, dtype=dtype).repeat(rows, 1)
    tokens = list(range(vocab)) * 2  # every id twice
    c = LogitControls(
        tokens=i32([tokens] * rows), lens=i32([len(tokens)] * rows),
        repetition=f32([v[0] for v in cases]), presence=f32([v[1] for v in cases]),
        frequency=f32([v[2] for v in cases]), bias_ids=i32(list(range(vocab)) * rows),
        bias_values=f32([v[3] for v in cases for _ in range(vocab)]),
        bias_starts=i32(np.arange(rows + 1) * vocab))
    got = control_logits(x.to(DEV), c).cpu().double().numpy()
    assert np.isfinite(got).all()
    for r, case in enumerate(cases):
        rep, pres, freq, bias = (float(np.float32(v)) for v in case)
        want = ref.control(x[r].double().numpy(), tokens, 0, rep, pres, freq,
                           [(i, bias) for i in range(vocab)], None)
        cut = np.clip(want, -most, most)
        size = np.abs(x[r].double().numpy()) * max(rep, 1 / rep) + abs(pres) + 2 * abs(freq) \
            + abs(bias)
        tol = torch.finfo(dtype).eps / 2 * np.abs(cut) + 5 * 2.0 ** -24 * np.minimum(
            size, 8 * 3.5e38)
        assert (np.abs(got[r] - cut) <= tol * (1 + 2.0 ** -7)).all(), (case, got[r], cut)
        assert (got[r][np.abs(want) > 1.01 * most] == cut[np.abs(want) > 1.01 * most]).all()
    # what is drawn from such a row is one of its ids
    out = control_logits(x.to(DEV), c)
    for temp in (0.0, 1e-3, 1.0, 3e38):
        st = torch.zeros(1, dtype=torch.int32, device=DEV)
        ids, _ = sample_each(out, f32([temp] * rows), status=st)
        assert int(st) == 0 and int(ids.min()) >= 0 and int(ids.max()) < vocab


def test_values_between_the_steps_are_not_cut_to_the_type():
    """Only the last rounding is the type's: 60000 / 0.5 passes fp16's 65504, less a
    presence of 1e5 it is 20000."""
    x = torch.tensor([[60000.0, 1.0]], dtype=torch.float16, device=DEV)
    c = LogitControls(tokens=i32([[0]]), lens=i32([1]), repetition=f32([0.5]), presence=f32([1e5]))
    assert control_logits(x, c)[0].tolist() == [20000.0, 1.0]
    c = LogitControls(tokens=i32([[0]]), lens=i32([1]), repetition=f32([0.5]),
                      bias_ids=i32([0, 1]), bias_values=f32([-1e5, 2.0]), bias_starts=i32([0, 2]))
    assert control_logits(x, c)[0].tolist() == [20000.0, 3.0]


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_finite_still_shows(dtype):
    x = torch.tensor([[1.0, -1.0, INF, -INF, float("nan"), 2.0]], dtype=dtype, device=DEV)
    tokens = [0, 1, 2, 3, 4] * 2

    def run(**kw):
        c = LogitControls(tokens=i32([tokens]), lens=i32([len(tokens)]),
                          **{k: f32([v]) for k, v in kw.items()})
        return control_logits(x, c)[0].tolist()

    out = run(presence=INF)      # never again
    assert out[:2] == [-INF, -INF] and np.isnan(out[2]) and out[3] == -INF and out[5] == 2.0
    out = run(frequency=-3e38)   # the penalty itself passes fp32
    assert all(np.isfinite(out[:2])) and out[2] == INF and out[3] == -INF and np.isnan(out[4])
    out = run(repetition=float("nan"))
    assert np.isnan(out[0]) and np.isnan(out[1])
    c = LogitControls(bias_ids=i32([0, 1, 2, 3, 4]), bias_values=f32([-INF, INF, 1, 1, 1]),
                      bias_starts=i32([0, 5]))
    out = control_logits(x, c)[0].tolist()
    assert out[:4] == [-INF, INF, INF, -INF] and np.isnan(out[4]) and out[5] == 2.0


@pytest.mark.parametrize("temperature", [1e37, 1e38, 3e38])
def test_top_k_of_logits_further_apart_than_fp32_reaches(temperature):
    """3e38 and -3e38 are 6e38 apart, which at such temperatures still weighs."""
    rows = 40
    u = (np.arange(rows) + 0.5) / rows
    x = torch.tensor([-3.3e38, 3e38, -3e38, 1.0, -3.2e38], dtype=torch.float32).repeat(rows, 1)
    for k in (1, 2, 3, 4):
        ids, _ = sample_each(x.to(DEV), f32([temperature] * rows), i32([k] * rows),
                             uniforms=f32(u))
        for r in range(rows):
            want, _, gap = ref.draw(x[r].double().numpy(), float(np.float32(temperature)), k, 1.0,
                                    0.0, float(np.float32(u[r])))
            if gap > 5 * 2.0 ** -43:
                assert int(ids[r]) == want, (k, r)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,lens", [
    (3, 50257, (4096, 4097, 8192)), (2, 3000, (5000, 20000)), (5, 40, (4095, 9000, 0, 12289, 1)),
    (33, 131072, (8192, 6000, 4500))])
def test_histories_of_several_rounds(rows, vocab, lens, dtype):
    print(f"[history] {rows} {vocab} {lens} {dtype}", flush=True)
    rng = np.random.default_rng([rows, vocab])
    lens = [lens[r % len(lens)] for r in range(rows)]
    cap = max(lens) + 3
    x = torch.from_numpy(rng.normal(0, 3, (rows, vocab))).to(dtype)
    tokens = np.where(rng.random((rows, cap)) < 0.5, rng.integers(0, max(1, vocab // 50), (rows, cap)),
                      rng.integers(0, vocab, (rows, cap)))
    prompt = [int(n * f) for n, f in zip(lens, rng.random(rows))]
    rep, pres, freq = 1.25, 0.5, 2.0 ** -7
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    c = LogitControls(tokens=i32(tokens), lens=i32(lens), prompt_lens=i32(prompt),
                      repetition=f32([rep] * rows), presence=f32([pres] * rows),
                      frequency=f32([freq] * rows))
    got = control_logits(x.to(DEV), c, status=st).cpu().double().numpy()
    assert int(st) == 0
    for r in range(rows):
        row, n, p = x[r].double().numpy(), lens[r], prompt[r]
        made = np.bincount(tokens[r, p:n], minlength=vocab)
        there = np.bincount(tokens[r, :n], minlength=vocab) > 0
        want = np.where(there, np.where(row > 0, row / rep, row * rep), row)
        want = want - np.where(made > 0, freq * made + pres, 0)
        size = np.abs(row) * rep + pres + freq * made
        tol = torch.finfo(dtype).eps / 2 * np.abs(want) + 4 * 2.0 ** -24 * size
        assert (np.abs(got[r] - want) <= tol * (1 + 2.0 ** -7)).all(), r
    # an id outside the vocabulary behind the first round is reported, too
    if max(lens) > 4200:
        r = lens.index(max(lens))
        tokens[r, 4150] = vocab
        c = LogitControls(tokens=i32(tokens), lens=i32(lens))
        control_logits(x.to(DEV), c, status=st)
        assert int(st) != 0

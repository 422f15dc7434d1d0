"""Branching decode (test_branch.py) where its definitions and its kernels'
short cuts could part: logits and scores that are no numbers, values that are
none and hardly weigh, starts that contradict themselves, lists and books
across layers, and numbers beyond their fields."""
import math

import pytest

from test_branch import plain_beams, run_beams, same_beams
from test_paged import dtypes

gpu = pytest.mark.gpu


@pytest.fixture
def torch_cuda():
    return pytest.importorskip("torch")


# ---------------------------------------------------------------------------
# beams


@gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [3, 40, 1025, 5003])
@pytest.mark.parametrize("n", [3, 33])
@pytest.mark.parametrize("case", ["all", "few left", "few left beside infinity", "-infinity among them", "one beam", "the end"])
def test_beam_select_nan_are_candidates(torch_cuda, kind, V, n, case):
    """NaN counts as -infinity: its token is chosen, the lowest first, where nothing better is left."""
    torch = torch_cuda
    B = 1 if case in ("few left", "few left beside infinity") else 2
    logits = torch.full((B, V), math.nan)
    scores = torch.tensor([[-1.0, -0.5][:B]])
    if case.startswith("few left"):
        logits[0, V // 2], logits[0, V - 1] = 1.0, 2.0
        if case == "few left beside infinity":  # (whatever lane has it has NaN too)
            logits[0, V // 3] = math.inf
    elif case == "-infinity among them":
        logits[0, ::2] = -math.inf
        logits[1, 1::2] = -math.inf
    elif case == "one beam":  # an ended beam beside it: one candidate
        logits[1, :] = 0.5
    elif case == "the end":
        logits[:, :2] = 1.0
    ended = torch.tensor([[0, 1]]) if case == "one beam" else None
    logits = logits.to(dtypes(torch)[kind])
    got = run_beams(torch, logits.cuda(), scores.cuda(), n, ended.to(torch.uint8).cuda() if ended is not None else None,
                    1 if ended is not None else -1)
    same_beams(got, plain_beams(torch, logits, scores, ended, 1 if ended is not None else -1, n))


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("low", [-math.inf, math.nan])
@pytest.mark.parametrize("V", [5, 3000, 70000])
def test_beam_select_ties_of_beams_without_a_score(torch_cuda, kind, low, V):
    """All tokens of a beam whose score is -infinity tie, whatever their logits: the lowest ones are chosen."""
    torch = torch_cuda
    g = torch.Generator().manual_seed(V)
    logits = torch.randn(8, V, generator=g).to(dtypes(torch)[kind])
    scores = torch.tensor([[-1.0, low, -2.0, low], [low, low, low, low]])
    ended = torch.tensor([[1, 0, 1, 0], [0, 1, 0, 0]])
    got = run_beams(torch, logits.cuda(), scores.cuda(), 12, ended.to(torch.uint8).cuda(), 4)
    same_beams(got, plain_beams(torch, logits, scores, ended, 4, 12))

"""The logarithm of beam selection's sums: rows whose rounding errors do not average out, and long runs per warp."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _check(logits, b, k, raises):
    """Scores of the best continuations against 64 bits.

    A term e^d, d = logit - reference, is off by |d| (2^-24 + 2^-24 + 2^-26) of its rounded argument (difference,
    product, log2 e) and by 2^-22 of the instruction; 7 sums in f32 add 7 * 2^-24.  The reference is at most 4 below the
    largest logit, and |d| counts by the terms' weights.  Each raise of it is off by 2^-22, and counts once more for the
    argument.  The result's own rounding is 2^-24 of it."""
    import smallaios_b200 as sa

    scores = torch.zeros(b, k, device=logits.device)
    parents, tokens, got = sa.beam_select(logits, scores, keep=k)
    lse, far = [], []
    for part in logits.split(256):
        x = part.double()
        top = x.amax(-1, keepdim=True)
        e = (x - top).exp()
        lse.append(top[:, 0] + e.sum(-1).log())
        far.append(((top - x) * e).sum(-1) / e.sum(-1))
    lse, far = torch.cat(lse), torch.cat(far)
    row = torch.arange(b, device=logits.device)[:, None] * k + parents.long()
    want = logits[row, tokens.long()].double() - lse[row]
    limit = (far[row] + 4 + 8 * (raises > 0)) * 2.25 * 2.0 ** -24 + (1 + raises) * 2.0 ** -22 + 7 * 2.0 ** -24
    off = (got.double() - want).abs() - 2.0 ** -24 * want.abs()
    assert (off <= limit).all(), f"{off.max().item():.2e} of {limit.min().item():.2e}"


def test_long_runs_that_climb_slowly(cuda_device):
    """4800 rows: a warp takes a whole one, and every step of it holds a logit above all before."""
    rows, v = 4800, 32768
    slope = 1e-5 * (0.7 + 0.1 * torch.arange(rows, device=cuda_device) % 0.7)
    logits = torch.arange(v, device=cuda_device, dtype=torch.float32) * slope[:, None]
    _check(logits, rows // 4, 4, 0)  # (less than 4 in all)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rest", [-3.0, -7.0, -9.7, -12.7])
def test_many_equal_logits_under_a_larger_one(cuda_device, rest, dtype):
    logits = torch.full((8, 128256), rest, device=cuda_device)
    logits[:, 5] = 0.3
    logits[4:, 70000] = 4.6  # in another step, or run
    _check(logits.to(DT[dtype]), 2, 4, 1)


@pytest.mark.parametrize("rows", [8, 4800])
def test_steps_and_equal_rows(cuda_device, rows):
    v = 32768
    for logits, raises in ((torch.zeros(rows, v, device=cuda_device), 0),
                           ((torch.arange(v, device=cuda_device) // 512 * 0.11).expand(rows, v).contiguous(), 2)):
        _check(logits, rows // 4, 4, raises)

"""balance_loss by sequence, in every type and for every form of a row: its
counts, loss and gradient against the definition in 64 bits."""
import pytest
import torch

from test_gpu_layer import DTYPES, _check_balance, _gen, _randn, _top

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


# experts: rows of whole vectors, 8 to 64 lanes of one and two vectors or more; and rows that are not
@pytest.mark.parametrize("E", [8, 32, 64, 128, 256, 512, 1024, 5, 63, 130, 255, 700])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_sequences_of_every_row_form(dtype, score, E):
    T, k = 333, min(E, 7)
    cuts = [4, 4, 5, 90, 90, 200, 201, 310]  # empty and single tokens among them, tokens of none at both ends
    logits = _randn((T, E), dtype, E, 1.5)
    ids = _top(logits, k)
    _check_balance(logits, ids, cuts, None, score)
    mask = torch.rand(T, generator=_gen(E), device="cuda") > 0.4
    mask[90:200] = False  # a sequence whose tokens are all left out
    logits[~mask] = float("nan")  # what a token that is left out holds
    _check_balance(logits, ids, cuts, mask, score)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_long_sequences(dtype):
    """Pieces of 16 waves, and sums by columns of experts."""
    T, E, k = 20000, 72, 6
    logits = _randn((T, E), dtype, 1, 1.5)
    mask = torch.rand(T, generator=_gen(2), device="cuda") > 0.2
    for cuts in ([0, T], [0, 7, 9000, 9000, T - 3]):
        _check_balance(logits, _top(logits, k), cuts, mask, "sigmoid")

"""Training operators where a call meets a limit of its kernels (GPU)."""

import pytest
import torch

from llm_hgemm import train_capi
from tests import training_reference as ref
from tests.gpu_helpers import require_cuda
from tests.test_gpu_training import loss_inputs, loss_through_c, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def _cuda():
    require_cuda()


@pytest.mark.parametrize("tokens, vocab, piece, tile", [
    (2049, 8256, 8192, 128), (3841, 4672, 4608, 256 | train_capi.TILE_PAIR), (8192, 9108, 0, 0),
], ids=["single", "pair", "chosen"])
def test_loss_short_last_piece_of_many_tile_rows(tokens, vocab, piece, tile):
    """At least 16 rows of tiles, where the raster's groups of rows depend on the
    sum's length: a last piece short enough for taller groups still adds each tile
    of dx to its own."""
    x, w, t = loss_inputs(tokens, 520, vocab, torch.bfloat16)
    dl = torch.tensor([64.0], device="cuda")
    want = ref.loss(x, w, t, "sum", -100, dl)
    got = loss_through_c(x, w, t, dl, tile, piece, train_capi.LOSS_SUM)
    for g, v in zip((got[0][0], got[1], got[2]), want):
        within(g, v)

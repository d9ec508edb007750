"""Tree and scored decode where two kernels, two tiles or two lengths meet, and with values that are no numbers."""
import random

import pytest
import torch

import cache_util as U
from test_gpu_decode_tree import _scored_case

pytestmark = pytest.mark.gpu

F, H = torch.float32, torch.bfloat16


@pytest.mark.parametrize("Hq,q_dtype,D", [(129, F, 128), (160, F, 64), (257, H, 128), (300, H, 64)])
def test_scores_of_more_heads_than_a_tile(Hq, q_dtype, D):
    """The query tiles of a KV head (128 rows, 256 of a bf16 q) are cut apart from one another."""
    rng = random.Random(Hq)
    _scored_case(41, [rng.randint(200, 4000) for _ in range(32)], Hq, 1, D, q_dtype, H, F, 0, 1.0)

"""linear_adapted at sizes that choose its 128 x 128 tiles (fp32 from 192 of them, bf16 from 384 of them to 192 of 256 x 256), and a
block of the model with adapters at the benchmark's batch, whose linear1 they are."""
import numpy as np
import pytest

import sequence_forms as F
from conftest import npy
from test_gpu_sequence import BLOCKS, assert_linear, block_adapters, linear_ref, merged, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def tiles(rows, M, t):
    return -(-rows // t) * -(-M // t)


@pytest.mark.parametrize("M", ["whole lines", "groups of four", "odd"])
@pytest.mark.parametrize("B, T, K, n, r", [(41, 100, 100, 5, 8), (4100, 1, 64, 70, 4), (2, 2061, 33, 3, 33), (33, 125, 136, 4, 128), (1, 4097, 500, 1, 16)], ids=str)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_linear_adapted_128_tiles(ops, dtype, B, T, K, n, r, M):  # noqa: F811
    """Tiles of one adapter, of several and of one a row; ragged rows, columns and K; outputs stored as lines, fours and one by one; x as
    a transposed view as well."""
    import torch
    M = {"whole lines": 1056, "groups of four": 1060, "odd": 1051}[M] if dtype == "float32" else {"whole lines": 1904, "groups of four": 1908, "odd": 1901}[M]
    assert tiles(B * T, M, 128) >= 192 if dtype == "float32" else tiles(B * T, M, 128) >= 384 and tiles(B * T, M, 256) < 192
    args = F.linear_inputs(3, B, T, K, M, n, r, getattr(torch, dtype))
    x, w, b, down, up, scale, ids = (t.cuda() for t in args)
    y = ops.linear_adapted(x, w, b, down, up, scale, ids)
    assert_linear(y, *linear_ref(x, w, b, down, up, scale, ids, False), K, r, dtype == "bfloat16")
    assert F.held(y.cpu(), F.linear_exact(*args), F.linear_fp32(*args)) <= 1
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    relu = ops.linear_adapted(turned, w, b, down, up, scale, ids, relu=True)
    assert torch.equal(relu, torch.relu(y))


@pytest.mark.parametrize("module", list(BLOCKS))
def test_block_of_the_model_with_adapters_at_the_benchmark_batch(ops, module):  # noqa: F811
    """256 sequences of up to 125 frames: linear1 with its padded weight rows and its frame-major output in the 128 tiles (H = 256: 250 x 2
    of them), linear2 in one launch."""
    import torch
    from mobileposer_amd import synthetic
    from oracle import mp_oracle as O
    weights = synthetic.make_weights(0)
    n_in, H, dirs, n_out = BLOCKS[module]
    B, T = 256, 125
    assert H < 256 or tiles(B * T, H, 128) >= 192
    adapters = block_adapters(module, 5, 4, 8, 50)
    dev = {k: tuple(t.cuda() for t in v) for k, v in adapters.items()}
    gen = torch.Generator().manual_seed(51)
    x = torch.randn(B, T, n_in, generator=gen)
    lengths = [max(1, T - 7 * (b % 18)) for b in range(B)]
    ids = [b % 6 - 1 for b in range(B)]
    y, (h, c) = ops.rnn_forward(module, x.cuda(), lengths, None, dev, ids)
    for b in (0, 1, 2, 100, 127, 128, 201, 255):
        a = None if ids[b] < 0 else ids[b]
        n = lengths[b]
        wy, (wh, wc) = O.rnn_forward(merged(weights, O.PREFIX[module], adapters, a), O.PREFIX[module], x[b:b + 1].numpy(), [n])
        assert np.abs(npy(y[b, :n]) - wy[0, :n]).max() < 1e-4
        assert np.abs(npy(h[:, b]) - wh[:, 0]).max() < 1e-4 and np.abs(npy(c[:, b]) - wc[:, 0]).max() < 1e-4

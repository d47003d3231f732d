"""The weight gradient of very many tokens: what the matrix units cut off does
not grow with them."""
import pytest
import torch

import act_ref as ref
import ark_b200 as ab

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def same_sign(tokens, nin, nout, dtype, seed):
    """All terms positive, so that a one-sided loss adds up; sums of about 2^-9 a token."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(8, 16, (tokens, nin), generator=g, device="cuda", dtype=torch.uint8)     # 4 bits: held exactly
    dy = (2.0 ** -8 + 2.0 ** -8 * torch.rand(tokens, nout, generator=g, device="cuda")).to(dtype)
    return (x.to(dtype) / 16), dy


def sums(x, dy):
    """64-bit sums, by parts of the tokens."""
    return sum(x[i: i + 16384].double().T @ dy[i: i + 16384].double() for i in range(0, x.shape[0], 16384))


# an addition of 16 tokens loses at most 2^-23 of the sum of magnitudes: 128 of them in an FP32
# gradient, 512 in an FP16 and 4096 in a BF16 one; the FP32 additions of the runs 2^-24 each
LOSS = {F32: 128 * 2.0 ** -23, F16: 512 * 2.0 ** -23, BF16: 4096 * 2.0 ** -23}


@pytest.mark.parametrize("tokens,nin,nout,dtype,out", [
    (131072, 2048, 2304, F16, F16),      # 72 tiles of 256 x 256, the tokens not split
    (131072, 2048, 2304, F16, F32),
    (128000, 4096, 256, BF16, F32),      # 16 tiles
    (128000, 4096, 256, BF16, BF16),
    (40001, 2048, 2301, BF16, BF16),     # odd
    (140000, 2048, 2304, BF16, BF16),
    (300000, 256, 256, F16, F32),        # one tile
])
def test_long_sums_keep_their_size(tokens, nin, nout, dtype, out):
    x, dy = same_sign(tokens, nin, nout, dtype, tokens)
    want = sums(x, dy)
    got = ab.weight_grad(ab.act8_pack(x, "int8"), dy, dtype=out)
    runs = tokens / 2048 + 16
    tol = ref.HALF[out] * want + (LOSS[out] + runs * 2.0 ** -24) * want
    off = (got.double() - want).abs()
    assert (off <= tol).all(), (off / want).max().item()
    if out != F32:       # added to what is there: two roundings to the type
        acc = got.clone()
        ab.weight_grad(ab.act8_pack(x, "int8"), dy, out=acc, accumulate=True)
        off = (acc.double() - got.double() - want).abs()
        assert (off <= ref.HALF[out] * 2 * want * 1.01 + (LOSS[out] + runs * 2.0 ** -24) * want).all()

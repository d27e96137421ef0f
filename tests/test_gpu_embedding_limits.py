"""pmg::embedding at the ends of what its arguments allow: padding ids counted from either end of the table."""
import pytest
import torch

from oracle import lm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('V', [1, 9, 3000])
def test_padding_counted_from_either_end(gpu, V):
    from paccmann_generator_amd import _ffi, ops
    torch.manual_seed(V)
    w = torch.randn(V, 12, device='cuda', requires_grad=True)
    ids = torch.cat([torch.arange(V), torch.randint(0, V, (50,))]).cuda()
    slope = torch.randn(len(ids), 12, device='cuda')
    for pad in {-V, -1, -(V // 2) - 1, V - 1, 0}:
        out = ops.embedding(w, ids, padding_idx=pad)
        assert torch.equal(out, w[ids])                      # the padding row is looked up like any other
        got, = torch.autograd.grad(out, w, slope)
        want, size, count = lm.embedding_grad(slope.cpu(), ids.cpu(), V, 1.0, pad % V)
        # a token's positions are added in fp32 (dropping the padding's positions moves where the sums are cut)
        assert bool(((got.cpu().double() - want).abs() <= size * (count.unsqueeze(1) + 2) * 2.0 ** -24).all()), pad
        assert not got[pad].any() and (V == 1 or bool(got.any(1).sum() == V - 1)), pad
    for pad in (V, -V - 1):
        with pytest.raises(_ffi.PmgError, match='padding_idx'):
            ops.embedding(w, ids, padding_idx=pad)


@pytest.mark.parametrize('dtype,E', [(torch.float32, 3), (torch.bfloat16, 8)], ids=str)
def test_more_positions_than_one_joining_launch_takes(gpu, dtype, E):
    """Narrow rows in chunks of 8 positions, more than 2^24 of them.  Every position adds small whole numbers, so that all
    partial sums are exact: a token's gradient is its number of positions times its row."""
    import paccmann_generator_amd  # noqa: F401  (registers the operators)
    N, V = (1 << 27) + 12345, 60001
    ids = torch.randint(0, V - 1, (N,), device='cuda', dtype=torch.int32, generator=torch.Generator(device='cuda').manual_seed(1))
    ids[-3000000:] = V - 1                     # a run over very many chunks, most of them of the last launch
    row = torch.tensor([1.0, -2.0, 3.0, 0.0, 4.0, -1.0, 2.0, 5.0][:E], device='cuda', dtype=dtype)
    got = torch.ops.pmg.embedding_bwd(row.repeat(N, 1), ids, V, 1.0, -1)
    count = torch.bincount(ids, minlength=V)
    want = count.double().unsqueeze(1) * row.double()
    assert int(count.max()) * 5 < 1 << 24      # whole numbers that fp32 holds
    assert torch.equal(got, want.to(dtype))


def test_more_rows_than_one_lookup_launch_takes(gpu):
    """138 GB of rows: every one of them is looked up."""
    from paccmann_generator_amd import ops
    N, V, E = (1 << 28) + 1001, 1000, 257
    if torch.cuda.mem_get_info()[0] < N * (E * 2 + 4) + (16 << 30):
        pytest.skip('needs 160 GB of free memory')
    table = torch.randn(V, E, device='cuda').bfloat16()
    ids = torch.randint(0, V, (N,), device='cuda', dtype=torch.int32)
    out = ops.embedding(table, ids, trusted_tokens=True)
    wrong = sum(int((out[n:n + (1 << 23)] != table[ids[n:n + (1 << 23)]]).any()) for n in range(0, N, 1 << 23))
    del out
    torch.cuda.empty_cache()
    assert wrong == 0

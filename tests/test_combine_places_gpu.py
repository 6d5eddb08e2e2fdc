"""The combine where choices belong to no expert (place -1): they add nothing, whatever the rows hold.

Tolerance as for the combine of k rows (test_combine_gpu.py): half a step of bf16 and 2^-19 of the sum of the terms' magnitudes; a piece
more is one more rounding of at most 17, within that."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pieces", [1, 2])
@pytest.mark.parametrize("left", [0.3, 1.0])
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 4, 4), (1, 6, 8, 256), (5, 2, 8, 260), (33, 3, 60, 132), (40, 8, 64, 1028), (300, 9, 64, 64), (200, 17, 32, 36)])
def test_combine_leaves_out_pairs_without_a_place(cuda, T, k, E, H, left, pieces):
    from promoe_amd import ops
    print(f"case combine_places T={T} k={k} E={E} H={H} left={left} pieces={pieces}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(T + k + H)
    idx = torch.topk(torch.randn(T, E, device=cuda, generator=gen), k, dim=1).indices.int()
    idx[torch.rand(T, k, device=cuda, generator=gen) < left] = -1
    d = ops.dispatch(idx.contiguous(), E)
    n = int((idx >= 0).sum())
    rows = torch.randn(pieces, T * k, H, device=cuda, generator=gen)
    rows[:, n:] = float("nan")                                    # (with all choices left out: every row, the first among them)
    w = torch.rand(T, k, device=cuda, generator=gen)
    w[idx < 0] = float("nan")
    shared = torch.randn(T, H, device=cuda, generator=gen)
    got = ops.combine(rows.view(-1, H), shared, w, d.pos_of_pair, None, T, H, k, routed_pieces=pieces)
    torch.cuda.synchronize()
    order = torch.sort(torch.where(idx < 0, E, idx).reshape(-1), stable=True).indices[:n]
    terms = rows[:, :n].double().sum(0) * w.reshape(-1)[order, None].double()
    want, mag = shared.double(), shared.double().abs()
    want, mag = want.index_add(0, order // k, terms), mag.index_add(0, order // k, terms.abs())
    assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * mag).all()
    got = ops.combine(rows.view(-1, H), None, w, d.pos_of_pair, None, T, H, k, routed_pieces=pieces)
    want, mag = want - shared.double(), mag - shared.double().abs()
    assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * mag + 2.0 ** -50).all()
    if left == 1.0:
        assert not got.any()


def test_leaving_a_choice_out_is_as_its_weight_being_zero(cuda):
    """From the dispatch through the sort of tokens to the combine: the same bits (adding zero changes none of a sum that is not -0)."""
    from promoe_amd import ops
    print("case combine_block", flush=True)
    T, k, E, H = 70, 4, 8, 256
    gen = torch.Generator(device=cuda).manual_seed(3)
    idx = torch.topk(torch.randn(T, E, device=cuda, generator=gen), k, dim=1).indices.int().contiguous()
    w = torch.rand(T, k, device=cuda, generator=gen)
    away = torch.rand(T, k, device=cuda, generator=gen) < 0.4
    x = torch.randn(T, H, device=cuda, generator=gen)
    full, part = ops.dispatch(idx, E), ops.dispatch(torch.where(away, -1, idx).int().contiguous(), E)
    a = ops.combine(ops.sort_tokens(x, full), None, torch.where(away, 0.0, w), full.pos_of_pair, None, T, H, k)
    b = ops.combine(ops.sort_tokens(x, part), None, w, part.pos_of_pair, None, T, H, k)
    torch.cuda.synchronize()
    assert torch.equal(a, b)

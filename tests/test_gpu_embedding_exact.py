"""Gradient of the embedding lookup on small whole numbers into float32: every partial sum is a whole number below 2^24, the
scale and beta are powers of two, so that the result is exact in any order, and one position lost or added twice shows.

A hot table row is added up in parts (its first chunk, whole workgroups of chunks, the chunks behind them), which depend on
where its positions begin and end among the sorted ones.  So it is laid one place before, on and behind the borders of chunks
and workgroups, for every number of teams that a workgroup can hold.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BETAS = (0.0, 1.0, 0.5)


def whole_numbers(n, d, t, cuda):
    i, c = torch.arange(n, device=cuda)[:, None], torch.arange(d, device=cuda)[None, :]
    return (1 + (7 * i + 3 * c) % 13).to(t)


def check(cuda, g, idx, rows, beta, what):
    from cagnet_amd import ops

    d = g.shape[1]
    old = (2 * (torch.arange(rows * d, device=cuda) % 7)).reshape(rows, d)
    inside = (idx >= 0) & (idx < rows)
    want = torch.zeros(rows, d, dtype=torch.int64, device=cuda).index_add_(0, idx[inside], g[inside].long()).double()
    want = want * 0.5 + (beta * old.double() if beta else 0.0)
    out = old.float() if beta else torch.full((rows, d), float("nan"), device=cuda)
    ops.embedding_bwd(g, idx, rows, 0.5, out=out, beta=beta)
    assert torch.equal(out.double(), want), what


def chunk_positions(n, d, t):
    """Sorted positions of a chunk, as the library cuts them: 8 to 512 by the number of indices, a quarter for narrow rows."""
    span = 8
    while span < 512 and span * span * 256 < n:
        span *= 2
    return max(span // 4, 8) if d * t.itemsize <= 128 else span


def teams_of(d, t):
    lanes = 1
    while lanes < -(-d * t.itemsize // 16) and lanes < 256:
        lanes *= 2
    return 256 // lanes


def light_rows(count, span):
    """Lengths of table rows that are not hot, `count` positions together."""
    out, k = [], 0
    while count > 0:
        out.append(min((span, 1, span - 1, 3, span)[k % 5], count))
        count -= out[-1]
        k += 1
    return out


def layout(start, end, n, span, second, outside):
    """Indices of n positions in sorted order: light rows up to `start`, a row from `start` to `end`, perhaps another right
    behind it of `second` positions, light rows, and `outside` positions that name no row."""
    lengths = light_rows(start, span) + [end - start] + ([second] if second else [])
    lengths += light_rows(n - outside - sum(lengths), span)
    idx = torch.repeat_interleave(torch.arange(len(lengths)) * 2 + 1, torch.tensor(lengths))  # every other row is not named
    rows = 2 * len(lengths) + 1
    return torch.cat([idx, torch.full((outside,), rows)]), rows


WIDTHS = [(torch.float32, d) for d in (3, 4, 7, 16, 30, 61, 128, 250, 511, 1000, 1030)] + \
    [(torch.bfloat16, d) for d in (5, 8, 13, 55, 261, 1000, 2056)] + [(torch.float16, d) for d in (32, 100)]


def test_widths_cover_every_number_of_teams():
    assert {teams_of(d, t) for t, d in WIDTHS} == {1, 2, 4, 8, 16, 32, 64, 128, 256}


@pytest.mark.parametrize("t,d", WIDTHS)
@pytest.mark.parametrize("least", [0, 4200, 20_000])  # the sort of one tile where n stays below 4097; longer chunks in the last
def test_hot_rows_at_the_borders_of_chunks_and_workgroups(cuda, t, d, least):
    teams, gen = teams_of(d, t), torch.Generator().manual_seed(d)
    span = chunk_positions(least, d, t)
    group = teams * span
    n = max(4 * group + 60, least)
    assert chunk_positions(n, d, t) == span
    g = whole_numbers(n, d, t, cuda)
    starts = sorted({group, group + min(3, teams - 1) * span})
    ends = sorted({group + min(5, teams) * span, 2 * group, 2 * group + min(3, teams - 1) * span, 3 * group, 4 * group - span})
    case = 0
    for s in starts:
        for e in ends:
            for ds in (-1, 0, 1):
                for de in (-1, 0, 1):
                    start, end = s + ds, e + de
                    case += 1
                    if end <= start or (least == 20_000 and case % 3):
                        continue
                    second = (0, span + 1, 0, min(group + 3, n - 6 - end))[case % 4]
                    idx, rows = layout(start, end, n, span, max(second, 0), 5 * (case % 2))
                    idx = idx[torch.randperm(n, generator=gen)].to(cuda)
                    check(cuda, g, idx, rows, BETAS[case % 3], (start, end, second, n))


@pytest.mark.parametrize("t,d", WIDTHS)
def test_hot_row_up_to_the_last_position(cuda, t, d):
    """The last table row is hot and ends with the array, or in front of positions that name no row."""
    teams, span = teams_of(d, t), 8
    group = teams * span
    gen = torch.Generator().manual_seed(d)
    for case, (start, end) in enumerate((a * group + b, c * group + e) for a in (0, 1) for b in (0, 1, span - 1)
                                        for c in (2, 3) for e in (-1, 0, 1, span)):
        for outside in (0, 7):
            n = end + outside
            lengths = light_rows(start, span) + [end - start]
            idx = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
            idx = torch.cat([idx, torch.full((outside,), -1)])[torch.randperm(n, generator=gen)].to(cuda)
            check(cuda, whole_numbers(n, d, t, cuda), idx, len(lengths), BETAS[case % 3], (start, end, outside))


@pytest.mark.parametrize("t,d", [(torch.float32, 3), (torch.float32, 33), (torch.float32, 128), (torch.bfloat16, 8),
                                 (torch.bfloat16, 300), (torch.float16, 41)])
@pytest.mark.parametrize("n", [4096, 70_000, 300_000])
def test_many_positions_of_one_row_and_of_popular_rows(cuda, t, d, n):
    gen = torch.Generator().manual_seed(n + d)
    g = whole_numbers(n, d, t, cuda)
    one = torch.full((n,), 4)
    third = torch.randint(0, 400, (n,), generator=gen)
    third[torch.rand(n, generator=gen) < 1 / 3] = 7
    popular = (410 ** torch.rand(n, generator=gen, dtype=torch.float64)).long() - 1
    popular[::50] = 410
    for idx in (one, third, popular):
        for beta in BETAS:
            check(cuda, g, idx.int().to(cuda), 410, beta, n)

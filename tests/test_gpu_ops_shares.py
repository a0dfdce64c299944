"""Tree attention of batches whose CTAs get more units than they write down at a time: long sequences set a CTA's share of the
tiles, and the short ones beside them fill another CTA's share with many units.  Against the definition in 64 bits (tolerances:
test_gpu_ops.attention)."""
import pytest
import torch

import qxops
from test_gpu_ops import DEV, TYPES, attention, check_tree, gen, ints, make_cache, near, random_tree

pytestmark = pytest.mark.gpu

TILE = 64                 # cache rows of a tile
LISTED = 32               # pieces a CTA writes down at a time


def shares(lens, nodes, group, kv_heads, block_rows, chain, ctas):
    """The tiles that each CTA looks at, of each piece it has: the units' tiles laid end to end, cut evenly; in a chain those
    that no row of the block sees are left out."""
    units = []                                                   # (tiles, tiles that are seen)
    for a, m in zip(lens, nodes):
        if not m:
            continue
        for block in range(-(-m * group // block_rows)):
            row_end = min(m * group, (block + 1) * block_rows)
            sees = min(a + m, a + (row_end - 1) // group + 1) if chain else a + m
            units += [(-(-(a + m) // TILE), -(-sees // TILE))] * kv_heads
    total = sum(t for t, _ in units)
    each, extra = (1, 0) if total < ctas else divmod(total, ctas)
    bounds = [each * c + min(c, extra) for c in range(min(ctas, total) + 1)]
    got, first, c = [[] for _ in bounds[1:]], 0, 0
    for tiles, seen in units:
        while c < len(got) and bounds[c] < first + tiles:
            if bounds[c + 1] > first:
                got[c].append(max(0, min(min(tiles, bounds[c + 1] - first), seen) - max(0, bounds[c] - first)))
            if bounds[c + 1] >= first + tiles:
                break
            c += 1
        if c < len(got) and bounds[c + 1] == first + tiles:
            c += 1
        first += tiles
    return got


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def run(kind, hd, group, n, long_rows, longs, short_lens, nodes, chain, block_rows, per_sm, pieces, dead=False):
    """`longs` sequences of long_rows rows (the first: a slot each), then the short ones, which share a slot."""
    g = gen(n + hd)
    c = make_cache(g, longs + 1, 1, long_rows + n, 1, hd)
    lens, slots = [long_rows] * longs + short_lens, list(range(longs)) + [longs] * len(short_lens)
    for k in per_sm:
        got = shares(lens, nodes, group, 1, block_rows, chain, k * sms())
        assert max(map(len, got)) > pieces
        if dead:
            assert any(len(x) > pieces and x[0] == 0 for x in got)
    q = torch.randn(len(lens), n, group, hd, generator=g, device=DEV).to(TYPES[kind])
    check_tree(c, 0, ints(slots), ints(lens), ints(nodes), q, None if chain else random_tree(len(lens), n, 5), hd ** -0.5,
               want_mass=False)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,chain,tiles,lists", [(64, True, 1, 3), (128, False, 1, 2), (64, False, 3, 2)])
def test_more_pieces_than_a_list_in_trees_on_tcgen05(kind, hd, chain, tiles, lists):
    """More than 32 and more than 64 pieces to a CTA, of one tile and of up to three."""
    n, shorts = 5, 2 * LISTED * lists                            # 40 query rows
    short_lens = [(i * 37) % (TILE * tiles - n) for i in range(shorts)]
    share = tiles * (LISTED * (lists - 1) + 8)
    longs = 2
    long_rows = TILE * -(-share * sms() // longs)
    run(kind, hd, 8, n, long_rows, longs, short_lens, [n] * longs + [1 + i % n for i in range(shorts)], chain, 128, (1,),
        LISTED * (lists - 1))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_first_piece_without_tiles_and_more_than_a_list_behind_it(kind):
    """A CTA that begins in a chain's tail which its first block of rows does not see, and goes on with two more lists."""
    n, group, hd, share = 40, 8, 64, 76
    # 40 nodes behind 30 rows: three blocks of two tiles, the first of which (nodes 0 to 15) sees one; the last CTA begins at its second
    shorts = share - 5
    lens, nodes = [30] + [(i * 11) % 40 for i in range(shorts)], [1, n] + [1 + i % 16 for i in range(shorts)]
    run(kind, hd, group, n, TILE * ((sms() - 1) * share - 1) - 1, 1, lens, nodes, True, 128, (1,), 2 * LISTED, dead=True)


@pytest.mark.parametrize("kind,hd,n,block_rows,per_sm", [("bf16", 64, 1, 16, (2, 3, 4)), ("f32", 64, 2, 16, (2, 3, 4)), ("f16", 128, 4, 32, (2,)),
                                                         ("f32", 64, 3, 32, (2,))])
@pytest.mark.parametrize("chain", [True, False])
def test_more_pieces_than_a_list_in_small_trees(kind, hd, n, block_rows, per_sm, chain):
    shorts = 3 * LISTED
    short_lens = [(i * 29) % (TILE - n) for i in range(shorts)]
    longs = 3
    long_rows = TILE * -(-(2 * LISTED + 6) * max(per_sm) * sms() // longs)
    run(kind, hd, 8, n, long_rows, longs, short_lens, [n] * longs + [1 + i % n for i in range(shorts)], chain, block_rows, per_sm,
        2 * LISTED)


@pytest.mark.parametrize("order", ["short first", "alternating"])
def test_a_batch_of_fresh_and_long_sequences(order):
    """64 trees of 16 nodes, half of the sequences at 20 rows and half at 4096, with weights; each as it is alone."""
    g = gen(64)
    seqs, n, ctx = 64, 16, 4096
    c = make_cache(g, seqs, 1, ctx + n, 4, 128)
    lens = [20] * 32 + [ctx] * 32 if order == "short first" else [20, ctx] * 32
    if order == "short first":
        assert max(map(len, shares(lens, [n] * seqs, 8, 4, 128, False, sms()))) > LISTED
    q = torch.randn(seqs, n, 32, 128, generator=g, device=DEV).bfloat16()
    slots, mask, status = torch.randperm(seqs, generator=g, device=DEV).to(torch.int32), random_tree(seqs, n, 2), ints([0])
    mass = torch.zeros_like(c.k_scales)
    out = qxops.tree_attention(c, 0, slots, ints(lens), q, mask=mask, mass=mass, status=status)
    assert int(status) == 0
    some = [0, 1, 31, 32, 62, 63]
    args = (slots[some], ints(lens)[some], ints([n] * len(some)), q[some], mask[some], 128 ** -0.5)
    w_out, _, w_mass, tol, _, tol_mass = attention(c, 0, *args)
    near(out[some], w_out, tol, "out")
    at = slots[some].long()
    near(mass[at], w_mass[at], tol_mass[at] + 2.0 ** -24 * w_mass[at], "mass")

"""shared_attention against attention in 64 bits over each sequence's own table."""
import numpy as np
import pytest

import affon_amd as A
from tests.drafts import NO_PAGE, Step, mask_words, set_tensor, stored, tree, upload

pytestmark = pytest.mark.gpu


def share(step, groups, shared):
    """The first shared[g] tokens of group g's sequences become its first one's:
    whole pages by the table, the rest as a copy."""
    per = step.B // groups
    for b in range(step.B):
        g = b // per
        first, s = g * per, int(shared[g])
        if b == first or step.lengths[b] < s:
            continue
        whole = s // step.page
        step.table[b, :whole] = step.table[first, :whole]
        for n in range(whole * step.page, s):
            (to, line), (page, from_line) = step.place(b, n), step.place(first, n)
            for cache in (step.keys, step.values):
                cache[:, to, :, line] = cache[:, page, :, from_line]
    return step


def run(session, step, shared, mask=None, **options):
    return A.shared_attention(step.cache, step.batch, upload(session, step.query, step.dtype),
                              upload(session, np.array(shared, np.uint32), "u32"),
                              None if mask is None else upload(session, mask_words(mask), "u32"), **options).storage()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 2), (128, 8, 2), (80, 5, 1), (96, 4, 4), (160, 4, 2), (256, 8, 1), (8, 2, 2)])
@pytest.mark.parametrize("T,masked,groups,own,shared", [
    (1, False, 1, (0, 5, 40, 63), (160,)), (1, False, 2, (7, 0, 70, 3), (64, 333)), (5, True, 1, (1, 90), (200,)),
    (40, True, 2, (3, 100), (130, 70))])
def test_shapes(session, rng, dtype, dim, heads, kv, T, masked, groups, own, shared):
    per = len(own) // groups
    lengths = [n + shared[b // per] for b, n in enumerate(own)]
    counts = [max(1, T - b % 3) for b in range(len(own))]
    step = share(Step(rng, B=len(own), T=T, heads=heads, kv=kv, dim=dim, lengths=lengths, counts=counts, dtype=dtype,
                      spread=2.0), groups, shared).device(session)
    mask = tree(rng, len(own), T) if masked else None
    step.check(run(session, step, shared, mask), mask)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,T,groups,shared,page", [(33, 1, 1, 2000, 16), (12, 7, 3, 1040, 48), (64, 1, 1, 5000, 64), (2, 1, 2, 700, 16)])
def test_many_sequences_and_long_prefixes(session, rng, dtype, B, T, groups, shared, page):
    shared = [shared - 128 * g for g in range(groups)]
    lengths = [shared[b // (B // groups)] + 17 * b % 130 for b in range(B)]
    step = share(Step(rng, B=B, T=T, heads=8, kv=2, lengths=lengths, page=page, dtype=dtype, spread=2.0), groups,
                 shared).device(session)
    step.check(run(session, step, shared))


@pytest.mark.parametrize("shared", [0, 1, 63, 64, 65, 127, 128, 4096, 0xFFFFFFFF])
def test_borders_of_the_prefix(session, rng, shared):
    """Prefixes that end anywhere, none, and ones that no sequence has."""
    lengths = [200, 128, 65, 64, 63, 0]
    step = Step(rng, B=6, T=2, lengths=lengths, spread=2.0)
    # All hold the longest's tokens, up to their own lengths: any prefix is shared.
    for b in range(1, 6):
        for n in range(lengths[b]):
            (to, line), (page, from_line) = step.place(b, n), step.place(0, n)
            for cache in (step.keys, step.values):
                cache[:, to, :, line] = cache[:, page, :, from_line]
    step.device(session)
    step.check(run(session, step, [shared]))


def test_sequences_that_do_not_share(session, rng):
    """The group's first has ended and its row of the table names others' pages; another is too short."""
    step = Step(rng, B=4, T=3, lengths=(0, 300, 310, 40), counts=(0, 3, 3, 2), spread=2.0)
    for n in range(256):
        (to, line), (page, from_line) = step.place(2, n), step.place(1, n)
        for cache in (step.keys, step.values):
            cache[:, to, :, line] = cache[:, page, :, from_line]
    step.device(session)
    table = step.table.copy()
    table[0] = rng.integers(0, step.pages + 9, step.table.shape[1])
    set_tensor(step.batch.page_table, table)
    got = run(session, step, [256])
    step.check(got)
    assert not got[:3].any()


def test_gaps_in_the_prefix_and_the_table(session, rng):
    step = share(Step(rng, B=3, T=2, lengths=(300, 290, 310), spread=2.0), 1, [256])
    step.table[:, 3] = NO_PAGE  # tokens 48 to 63 lie nowhere
    step.table[1, 18] = 0x7FFFFFFF
    step.device(session)
    step.check(run(session, step, [256]))


def test_layers_scales_and_outputs(session, rng):
    step = share(Step(rng, B=4, T=2, heads=8, layers=3, lengths=(150, 140, 133, 200)), 1, [130]).device(session)
    for scale in (-0.3, 0.0, 1.5):
        step.check(run(session, step, [130], layer=2, scale=scale), scale=scale, layer=2)
    query = upload(session, step.query, "bf16")
    shared = upload(session, np.array([130], np.uint32), "u32")
    out = A.shared_attention(step.cache, step.batch, query, shared, layer=1, out=query)
    assert out is query
    step.check(out.storage(), layer=1)


def test_odd_strides(session, rng):
    step = share(Step(rng, B=4, T=2, heads=4, lengths=(150, 140, 133, 200), spread=2.0), 2, [130, 64]).device(session)
    wide = np.zeros((8, 4 * 64 + 3), np.uint16)
    wide[:, 1:-2] = step.query
    query = A.slice(upload(session, wide, "bf16"), [{}, {"start": 1, "stop": 4 * 64 + 1}])
    shared = upload(session, np.array([130, 64], np.uint32), "u32")
    step.check(A.shared_attention(step.cache, step.batch, query, shared).storage())


def test_infinities_and_nans(session, rng):
    """NaN queries of rows not in use, and values that only some drafted rows see."""
    step = share(Step(rng, B=3, T=3, lengths=(200, 210, 190), counts=(3, 1, 2), spread=2.0), 1, [128])
    step.query[4] = step.query[5] = 0x7FC0
    page, line = step.place(0, 202)  # drafted token 2 of the first, which the last row alone sees
    step.values[0, page, 0, line, 3] = 0x7F80
    step.device(session)
    got = run(session, step, [128])
    step.check(got, rows=[0, 1, 3, 6, 7])
    head = got[2].view(np.uint16).reshape(4, 64)
    assert head[0, 3] == 0x7F80 and not got[4].any() and not got[5].any()


def test_it_is_tree_attention(session, rng):
    """Beside tree_attention of the same call: f32 sums in another order."""
    step = share(Step(rng, B=8, T=4, heads=8, kv=2, dim=128, lengths=[640 + 9 * b for b in range(8)], dtype="f32",
                      spread=2.0), 2, [640, 600]).device(session)
    query = upload(session, step.query, "f32")
    shared = upload(session, np.array([640, 600], np.uint32), "u32")
    plain = A.tree_attention(step.cache, step.batch, query).storage()
    got = A.shared_attention(step.cache, step.batch, query, shared).storage()
    step.check(got)
    step.check(plain)


def copies(rng, B, T, tokens, own, **options):
    """Sequences whose first `tokens` are the first one's, each with `own` more."""
    return share(Step(rng, B=B, T=T, lengths=[tokens + n for n in own], spread=2.0, **options), 1, [tokens])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("B,T,heads,kv,tokens,page", [
    (17, 1, 8, 2, 64, 16), (18, 2, 4, 2, 128, 16), (5, 9, 2, 1, 1000, 48), (9, 4, 16, 2, 640, 80), (30, 3, 4, 1, 2048, 64),
    (3, 30, 8, 1, 9000, 256), (33, 1, 2, 1, 17000, 64)])
def test_many_rows(session, rng, dim, B, T, heads, kv, tokens, page):
    """From 65 to hundreds of rows over a prefix, of several thousand keys to a workgroup too."""
    own = [(13 * b) % 31 for b in range(B)]
    step = copies(rng, B, T, tokens, own, heads=heads, kv=kv, dim=dim, page=page).device(session)
    for scale in (None, -0.1):
        step.check(run(session, step, [tokens], scale=scale), scale=scale)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("missing", [[0], [3, 4], [1, 2, 3], [8], list(range(12)), list(range(1, 12, 2))])
@pytest.mark.parametrize("page", [16, 48])
def test_gaps_under_many_rows(session, rng, dim, missing, page):
    """An odd number of 16-key tiles too, infinities and NaNs in the pages that lie behind."""
    step = copies(rng, 20, 1, 12 * page, [3 * b for b in range(20)], heads=8, kv=2, dim=dim, page=page)
    step.table[:, missing] = NO_PAGE
    step.device(session)
    step.check(run(session, step, [12 * page]))


def test_peaks_that_move(session, rng):
    """Scores that grow along the prefix: every row's reference moves many times."""
    step = copies(rng, 24, 1, 1024, [5] * 24, heads=4, kv=1, dim=128)
    query = stored(np.full((24, 4 * 128), 1.0) + rng.standard_normal((24, 4 * 128)) * 0.1, "bf16")
    step.query = query
    for n in range(1024):
        page, line = step.place(0, n)
        for b in range(24):
            step.keys[0, step.table[b, n // 16], :, line] = stored(np.full(128, n / 64.0), "bf16")
    step.device(session)
    step.check(run(session, step, [1024]))


@pytest.mark.parametrize("value", [0x7F80, 0xFF80, 0x7FC0])
def test_committed_values_that_are_not_finite(session, rng, value):
    """They reach every row, as the formula has it: infinities as such, NaN as NaN."""
    step = copies(rng, 20, 1, 256, [2] * 20, heads=8, kv=2, dim=64)
    page, line = step.place(0, 100)
    step.values[0, page, 1, line, 7] = value
    step.device(session)
    got = run(session, step, [256]).reshape(20, 8, 64)
    # Head 4 is the first of key head 1.
    odd = got[:, 4:, 7]
    assert (odd == value).all() if value != 0x7FC0 else ((odd & 0x7FFF) > 0x7F80).all()
    finite = got.copy()
    finite[:, 4:, 7] = 0
    assert ((finite & 0x7F80) != 0x7F80).all()


def test_odd_strides_of_many_rows(session, rng):
    step = copies(rng, 20, 1, 320, [9] * 20, heads=8, kv=2, dim=128).device(session)
    wide = np.zeros((20, 8 * 128 + 3), np.uint16)
    wide[:, 1:-2] = step.query
    query = A.slice(upload(session, wide, "bf16"), [{}, {"start": 1, "stop": 8 * 128 + 1}])
    step.check(A.shared_attention(step.cache, step.batch, query, upload(session, np.array([320], np.uint32), "u32")).storage())

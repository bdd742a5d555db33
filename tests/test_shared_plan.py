"""The host planner of the attention behind one shared prefix, on the CPU: every key that a row sees is
visited once, by an item inside its bounds, and every row is written once."""
import numpy as np
import pytest

import shared_ref as ref

FAKE, OUT = 0x100000, 0x200000  # aligned stand-in device addresses
TILE, ROWS = {0: 128, 1: 128, 2: 32}, {0: 256, 1: 128, 2: 16}


def make(qattn, prefix, queries, own, heads=16, kv=8, dim=128, page=64, paged=True, mask=0, always=176, window=432,
         form=0, rng=None, **kw):
    rng = rng or np.random.default_rng(0)
    need = [-(-prefix // page)] + ([-(-n // page) for n in own] if paged else [])
    pages = max(sum(need), 1) + 3
    order = rng.permutation(pages).astype(np.int32)
    cache = qattn.make_kv_cache(FAKE, FAKE, pages, page, kv, dim, format=form, k_scale=FAKE, v_scale=FAKE)
    return qattn.make_shared_desc(FAKE, OUT, cache, np.concatenate([[0], np.cumsum(queries)]), own, q_heads=heads,
                                  prefix_pages=order[:need[0]], prefix_len=prefix,
                                  own_pages=order[need[0]:sum(need)] if paged else None, k=None if paged else FAKE,
                                  v=None if paged else FAKE, mask=mask, prefix=always, window=window, **kw), order, need


def check_plan(qattn, prefix, queries, own, heads=16, kv=8, page=64, paged=True, mask=0, always=176, window=432, **kw):
    desc, order, need = make(qattn, prefix, queries, own, heads, kv, page=page, paged=paged, mask=mask, always=always,
                             window=window, **kw)
    plan, info = qattn.shared_plan(desc)
    group, T = heads // kv, int(np.sum(queries))
    seq = np.repeat(np.arange(len(queries)), queries)
    own = np.asarray(own, np.int64)
    position = np.concatenate([prefix + n - m + np.arange(m) for m, n in zip(queries, own)] + [np.zeros(0)]).astype(np.int64)
    assert np.array_equal(plan["positions"], np.maximum(position, -1))
    # groups of 16 keys in page order, each source's filled up to whole tiles
    tables = np.split(order[:sum(need)], np.cumsum(need)[:-1])
    groups, first_group = [], []
    for table, n in zip(tables, [prefix] + (list(own) if paged else [])):
        first_group.append(len(groups))
        k = np.arange(0, n, 16)
        groups += list((table[k // page] * kv * page + k % page) // 16)
        groups += [groups[-1]] * (-len(groups) % 8) if n else []
    assert np.array_equal(plan["groups"], groups)
    first_row = np.concatenate([[0], np.cumsum(own)])
    top = prefix + int(own.max(initial=0))
    counts = np.zeros((T * group, max(top, 1)), np.int16)  # visits of (row, key position)
    writes, parts, flat = np.zeros(T * group, int), {}, 0
    for it in plan["items"]:
        row0, rows, s0, s1, part, tiles, kind, least, greatest = it[:9]
        assert 1 <= rows <= ROWS[kind] and 0 <= row0 and row0 + rows <= T * group and tiles >= 1
        r = np.arange(row0, row0 + rows)
        at = plan["positions"][r // group]
        assert least <= at.min() and greatest >= at.max()
        segs = plan["segments"][s0:s1]
        assert sum(s[6] - s[5] for s in segs) == tiles and s1 > s0
        assert np.array_equal(it[12:24], segs[0])
        group_at = lambda s, k: 0 if s[0] == 2 else groups[s[2] + k // 16]  # noqa: E731
        visits = [(s0 + i, s, t) for i, s in enumerate(segs) for t in range(s[5], s[6])]
        if kind == 2:
            runs, done = plan["runs"][8 * flat:8 * flat + 8], 0
            flat += 1
            assert (runs[:, 10] <= -(-tiles // 8)).all() and runs[:, 10].sum() == tiles
            for run in runs[runs[:, 10] > 0]:
                i, s, t = visits[done]
                assert run[5] == t and run[9] == i and np.array_equal(np.delete(run[:9], 5), np.delete(s[:9], 5))
                assert list(run[11:13]) == [group_at(s, 32 * t), group_at(s, 32 * t + 16)]
                done += run[10]
        else:
            assert list(it[24:]) == [group_at(segs[0], 128 * segs[0][5] + 16 * i) for i in range(8)]
        for source, whole, base, keys, pos0, t0, t1, lo, hi in segs[:, :9]:
            assert 0 <= t0 < t1 <= -(-keys // TILE[kind])
            assert row0 <= lo < hi <= row0 + rows
            if source == 0:
                assert base == 0 and keys == prefix and pos0 == 0
                sees = np.ones(rows, bool)
            else:
                i = seq[lo // group]
                assert (seq[np.arange(lo, hi) // group] == i).all() and keys == own[i] and pos0 == prefix
                assert base == (first_group[1 + i] if paged else first_row[i]) and source == (1 if paged else 2)
                sees = (r >= lo) & (r < hi)
            key = np.arange(t0 * TILE[kind], min(t1 * TILE[kind], keys))
            counts[np.ix_(r[sees], pos0 + key)] += 1
            if whole:
                assert sees.all() and t1 * TILE[kind] <= keys
                assert all(ref.visible(position[x // group], pos0 + t1 * TILE[kind], mask, always, window)[pos0 + key].all()
                           for x in r)
        if part < 0:
            writes[r] += 1
        else:
            for j in range(rows):
                assert part + j not in parts and 0 <= part + j < info.partial_rows
                parts[part + j] = row0 + j
    assert len(plan["runs"]) == 8 * flat
    used = set()
    for m in plan["merges"]:
        writes[m[0]] += 1
        for first, count, step in (m[1:4], m[4:7]):
            for k in range(count):
                assert parts[first + k * step] == m[0] and first + k * step not in used
                used.add(first + k * step)
    assert used == set(parts) and (writes == 1).all()
    pairs = 0
    for row in range(T * group):
        t = row // group
        keep = ref.visible(position[t], prefix + own[seq[t]], mask, always, window)
        visits = counts[row, :len(keep)]
        assert (visits[keep] == 1).all() and (visits <= 1).all() and not counts[row, len(keep):].any()
        pairs += int(keep.sum()) if row % group == 0 else 0
    assert (info.tokens, info.pairs, info.flops) == (T, pairs, 4 * 128 * heads * pairs)
    assert info.keys == prefix + own.sum() and info.items == len(plan["items"])
    return plan, info


CASES = [
    dict(prefix=0, queries=[1], own=[1]),
    dict(prefix=0, queries=[1], own=[0]),                 # sees nothing
    dict(prefix=0, queries=[3], own=[1]),                 # two rows at positions below 0
    dict(prefix=1, queries=[1], own=[0]),
    dict(prefix=5, queries=[9], own=[2]),
    dict(prefix=0, queries=[0, 4, 0], own=[3, 4, 0]),     # sequences without queries
    dict(prefix=20, queries=[0, 0], own=[3, 0]),          # no queries at all
    dict(prefix=64, queries=[1] * 16, own=[1] * 16),
    dict(prefix=500, queries=[1] * 16, own=list(range(16)), page=16),
    dict(prefix=3000, queries=[1] * 64, own=[37 * i % 601 for i in range(64)]),
    dict(prefix=700, queries=[1] * 8, own=[1500, 700, 33, 1, 64, 65, 63, 0], heads=28, kv=4, page=32),
    dict(prefix=129, queries=[1] * 3, own=[10, 20, 30], heads=5, kv=5),
    dict(prefix=300, queries=[2, 1, 5, 8, 9, 1], own=[40, 50, 5, 8, 100, 1000]),
    dict(prefix=500, queries=[36, 84, 150, 10, 121, 67], own=[36, 84, 150, 10, 121, 67], paged=False),
    dict(prefix=1000, queries=[200, 1, 130, 7, 64], own=[250, 900, 130, 7, 164], heads=12, kv=4),
    dict(prefix=0, queries=[300, 1, 40], own=[300, 500, 40], paged=False),
    dict(prefix=130, queries=[300], own=[300], heads=64, kv=1),
    dict(prefix=700, queries=[50], own=[50], heads=3, kv=1, paged=False),
]


@pytest.mark.parametrize("mask,always,window", [(0, 0, 0), (1, 176, 432), (1, 0, 33), (1, 100, 1), (1, 64, 0), (1, 0, 0)])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_plan_visits_every_seen_key_once(qattn, case, mask, always, window):
    check_plan(qattn, mask=mask, always=always, window=window, **case)


def test_plans_of_random_batches(qattn):
    rng = np.random.default_rng(3)
    for _ in range(60):
        n = int(rng.integers(1, 12))
        queries = rng.choice([0, 1, 1, 2, 7, 8, 9, 30, 64, 65, 130], n)
        own = queries + rng.choice([0, 0, 1, 40, 300], n) - rng.choice([0, 0, 0, 1], n)
        heads, kv = [(16, 8), (4, 1), (6, 2), (3, 3)][rng.integers(4)]
        check_plan(qattn, int(rng.choice([0, 1, 31, 64, 100, 257, 900])), queries, np.maximum(own, 0), heads, kv,
                   page=int(rng.choice([16, 64, 128])), paged=bool(rng.integers(2)), mask=int(rng.integers(2)),
                   always=int(rng.choice([0, 20, 176])), window=int(rng.choice([1, 64, 100, 432])))


def test_plan_fills_the_chip_for_few_rows(qattn):
    # 64 tokens behind 8,192 keys, cut until most of the 32 slots of a KV head have work
    plan, _ = qattn.shared_plan(make(qattn, 8192, [1] * 64, [200] * 64)[0])
    assert len(plan["items"]) >= 24
    # a full batch fills it too
    _, info = qattn.shared_plan(make(qattn, 5000, [500] * 16, [500] * 16, paged=False)[0])
    assert info.items * 8 >= 400
    # masks skip whole tiles of the prefix
    plan, _ = qattn.shared_plan(make(qattn, 8192, [100], [100], mask=1)[0])
    blocks = {}
    for it in plan["items"]:
        blocks[it[0]] = blocks.get(it[0], 0) + it[5] * TILE[it[6]]
    assert max(blocks.values()) <= (2 + 6 + 2) * 128


def refuses(qattn, needle, change, **kw):
    case = dict(prefix=100, queries=[3, 1], own=[5, 70], **kw)
    desc, _, _ = make(qattn, **case)
    change(desc)
    with pytest.raises(qattn.QattnError) as e:
        qattn.shared_plan(desc)
    assert e.value.code == qattn.EINVAL and needle in str(e.value)


@pytest.mark.parametrize("needle,change,kw", [
    ("q/o", lambda d: setattr(d, "q", None), {}),
    ("q/o", lambda d: setattr(d, "o", FAKE + 8), {}),
    ("o is q", lambda d: setattr(d, "o", d.q), {}),
    ("o is q", lambda d: (setattr(d, "v", FAKE + 64), setattr(d, "o", FAKE + 64)), dict(paged=False)),
    ("row strides (q", lambda d: setattr(d, "q_row_stride", 2040), {}),
    ("row strides (q", lambda d: setattr(d, "o_row_stride", 2052), {}),
    ("row strides (q", lambda d: setattr(d, "q_row_stride", 1 << 25), {}),
    ("row strides (k", lambda d: setattr(d, "v_row_stride", 1016), dict(paged=False)),
    ("k/v NULL", lambda d: setattr(d, "k", None), dict(paged=False)),
    ("q_heads", lambda d: setattr(d, "q_heads", 12), {}),
    ("q_heads", lambda d: setattr(d, "q_heads", 0), {}),
    ("q_heads", lambda d: setattr(d, "q_heads", 8 * 65), {}),
    ("head_dim", lambda d: setattr(d.cache, "head_dim", 80), {}),
    ("page_size", lambda d: setattr(d.cache, "page_size", 24), {}),
    ("cache k/v", lambda d: setattr(d.cache, "v", None), {}),
    ("k_scale", lambda d: setattr(d.cache, "v_scale", None), dict(form=1)),
    ("mask", lambda d: setattr(d, "mask", 2), {}),
    ("window", lambda d: setattr(d, "window", -1), dict(mask=1)),
    ("scale", lambda d: setattr(d, "scale", -1.0), {}),
    ("scale", lambda d: setattr(d, "scale", float("nan")), {}),
    ("cu_seqlens", lambda d: setattr(d, "cu_q", None), {}),
    ("own_len", lambda d: setattr(d, "own_len", None), {}),
    ("prefix_len", lambda d: setattr(d, "prefix_len", -1), {}),
    ("prefix_len", lambda d: setattr(d, "prefix_len", 1 << 30), {}),
    ("prefix_pages", lambda d: setattr(d, "prefix_pages", None), {}),
    ("nseq", lambda d: setattr(d, "nseq", 0), {}),
    ("pages[", lambda d: setattr(d.cache, "pages", 2), {}),
    ("own_len[1]", lambda d: d._arrays[2].__setitem__(1, -1), {}),
    ("own_len[0]", lambda d: d._arrays[2].__setitem__(0, (1 << 30) - 100), dict(paged=False)),
    ("prefix_pages[0]", lambda d: d._arrays[0].__setitem__(0, -1), {}),
    ("own_pages[1]", lambda d: d._arrays[3].__setitem__(1, 1 << 20), {}),
    ("non-decreasing", lambda d: d._arrays[1].__setitem__(1, 9), {}),
])
def test_refusals(qattn, needle, change, kw):
    refuses(qattn, needle, change, **kw)


def test_refuses_too_many_rows_and_counts_pages(qattn):
    with pytest.raises(qattn.QattnError) as e:
        qattn.shared_plan(make(qattn, 0, [1 << 22], [5])[0])
    assert "2^22" in str(e.value)
    cache = qattn.make_kv_cache(FAKE, FAKE, 9, 64)
    with pytest.raises(ValueError):  # the binding: a list too short to be read
        qattn.make_shared_desc(FAKE, OUT, cache, [0, 1], [65], own_pages=[1])
    with pytest.raises(ValueError):
        qattn.make_shared_desc(FAKE, OUT, cache, [0, 1], [65, 3], own_pages=[1, 2, 3])
    # pages are not needed, nor looked at, where no page is read
    qattn.shared_plan(qattn.make_shared_desc(FAKE, OUT, qattn.make_kv_cache(None, None, 0, 0), [0, 2], [2], k=FAKE, v=FAKE))


def test_plans_of_the_longest_contexts(qattn):
    """One token behind nearly 2^30 cached keys, on pages that repeat: the plan covers them, in time."""
    prefix, page = (1 << 30) - 200, 4096
    n = -(-prefix // page)
    cache = qattn.make_kv_cache(FAKE, FAKE, 7, page, 1, 128, format=1, k_scale=FAKE, v_scale=FAKE)
    for queries, group in ((1, 1), (40, 4)):
        desc = qattn.make_shared_desc(FAKE, OUT, cache, [0, queries], [queries], q_heads=group, prefix_pages=np.arange(n) % 7,
                                      prefix_len=prefix, own_pages=[3])
        plan, info = qattn.shared_plan(desc)
        keys = sum(int(i[5]) * TILE[i[6]] for i in plan["items"])
        assert prefix <= keys <= (prefix + 4 * 128 + len(plan["items"]) * 32) * -(-queries * group // 16)
        assert info.pairs == sum(prefix + i + 1 for i in range(queries))
        assert int(plan["segments"][:, 6].max()) * 128 >= prefix and (plan["segments"][:, 5:7] >= 0).all()


def test_plans_of_many_sequences_in_time(qattn):
    import time
    desc = make(qattn, 2000, [1] * 4000, [1 + 37 * i % 300 for i in range(4000)])[0]
    start = time.time()
    plan, info = qattn.shared_plan(desc)
    assert info.tokens == 4000 and time.time() - start < 5

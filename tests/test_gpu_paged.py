"""Paged decoding on the GPU (estts_page_plan, estts_page_write, estts_paged_attention) against plain restatements: the plan in whole
numbers, the write bit for bit, the attention in float64 with bounds derived from the arithmetic (see attention_bound)."""
import ctypes
import math

import pytest
import torch

import estts
from estts import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda'
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


# ----------------------------------------------------------------------------------------------------------------- plan
def plan_oracle(lengths, new, table, free, n_free, page, T=None, R=None):
    """The rules of the header, one request after another."""
    B, P = len(lengths), len(table[0])
    lengths, table, free = list(lengths), [list(r) for r in table], list(free)
    cap = P * page
    lengths = [min(max(n, 0), cap) for n in lengths]
    pages = lambda n: -(-n // page)
    top = min(max(n_free, 0), len(free))
    for b in range(B):
        if new[b] < 0:
            for j in range(pages(lengths[b])):
                if top < len(free):
                    free[top] = table[b][j]
                    top += 1
    total = T if R is None else B * R
    slots, positions = [-1] * total, [-1] * total
    out, asked, taken, refused, start = list(lengths), 0, 0, 0, 0
    for b in range(B):
        want, first = max(new[b], 0), start
        start += want
        if new[b] < 0:
            out[b] = 0
            continue
        room = want == 0 or (want <= R if R is not None else start <= T)
        fits = room and lengths[b] + want <= cap
        need = pages(lengths[b] + want) - pages(lengths[b]) if fits else 0
        asked += need
        if not fits or (need and asked > top):
            refused += 1
            continue
        for i in range(need):
            table[b][pages(lengths[b]) + i] = free[top - 1 - taken]
            taken += 1
        out[b] = lengths[b] + want
        for i in range(want):
            r = first + i if R is None else b * R + i
            pos = lengths[b] + i
            page_id = table[b][pos // page]
            positions[r] = pos
            slots[r] = page_id * page + pos % page if 0 <= page_id < len(free) else -1
    return dict(slots=slots, positions=positions, table=table, free=free, lengths=out, n_free=top - taken, refused=refused)


def dev(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def run_plan(lengths, new, table, free, n_free, page, T=None, R=None, in_place=False):
    B = len(lengths)
    d = dict(lengths=dev(lengths), new=dev(new), block_table=dev(table), free_pages=dev(free), n_free=dev([n_free]))
    slots = torch.full((B, R) if R is not None else (T,), 77, dtype=torch.int32, device=DEV)
    positions, refused = torch.full_like(slots, 77), dev([77])
    lo, no = (None, None) if in_place else (dev([77] * B), dev([77]))
    ops.page_plan(page=page, slots=slots, positions=positions, lengths_out=lo, n_free_out=no, refused=refused, **d)
    if not in_place:
        assert d['lengths'].tolist() == list(lengths) and d['n_free'].item() == n_free
    return dict(slots=slots.view(-1).tolist(), positions=positions.view(-1).tolist(), table=d['block_table'].tolist(), free=d['free_pages'].tolist(),
                lengths=(d['lengths'] if in_place else lo).tolist(), n_free=(d['n_free'] if in_place else no).item(), refused=refused.item())


def random_state(B, P, page, longest, g):
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    lengths = [min(r(0, longest), P * page) for _ in range(B)]
    used = [-(-n // page) for n in lengths]
    extra = r(0, 2 * B)
    ids = torch.randperm(sum(used) + extra + 1, generator=g).tolist()
    table, at = [], 0
    for u in used:
        table.append(ids[at:at + u] + [-5] * (P - u))
        at += u
    free = ids[at:] + [-9] * at
    return lengths, table, free, len(ids) - at


@pytest.mark.parametrize('B', [1, 2, 63, 64, 65, 1000, 1024, 1025, 2500])
@pytest.mark.parametrize('page,longest,prompt', [(16, 90, 1), (16, 40, 70), (48, 300, 200)])
@pytest.mark.parametrize('layout', ['packed', 'padded'])
def test_page_plan_matches_the_rules(B, page, longest, prompt, layout):
    g = torch.Generator().manual_seed(B * 7 + page + prompt)
    P = -(-(longest + prompt) // page)
    lengths, table, free, n_free = random_state(B, P, page, longest, g)
    kind = torch.randint(0, 8, (B,), generator=g).tolist()
    new = [-1 if k == 0 else 0 if k == 1 else int(torch.randint(1, prompt + 1, (1,), generator=g)) for k in kind]
    rows = sum(max(n, 0) for n in new)
    # packed maps one entry too short for the last rows, padded ones too narrow for the longest prompts
    size = dict(T=max(1, rows - 1 if B % 2 else rows + 5)) if layout == 'packed' else dict(R=max(1, prompt - (B % 3)))
    want = plan_oracle(lengths, new, table, free, n_free, page, **size)
    for in_place in (False, True):
        got = run_plan(lengths, new, table, free, n_free, page, in_place=in_place, **size)
        for k in want:
            assert got[k] == want[k], (k, in_place)


@pytest.mark.parametrize('case', ['no pages', 'all end', 'nothing comes', 'lengths out of range', 'stack out of range', 'ids out of range', 'ended twice',
                                  'huge request'])
def test_page_plan_at_the_edges(case):
    page, P = 16, 3
    lengths, table, free, n_free = [20, 0, 48, 7], [[3, 1, -1], [-1, -1, -1], [0, 2, 4], [5, -1, -1]], [6, 7, 8, 0, 0, 0, 0, 0, 0], 3
    new = [1, 1, 0, 30]
    if case == 'no pages':
        n_free, new = 0, [1, 1, 1, 9]              # request 0 and 3 have room in a page, 1 needs one, 2 is at the end of its table row
    elif case == 'all end':
        new = [-1, -7, -1, -1]
    elif case == 'nothing comes':
        new = [0, 0, 0, 0]
    elif case == 'lengths out of range':
        lengths, new = [-4, 0, 99, 2 ** 31 - 1], [3, 0, 1, -1]
        table[3] = [5, 6, 7]
    elif case == 'stack out of range':
        n_free = 2 ** 30
    elif case == 'ids out of range':
        table[0][1], free[2], new = 2 ** 20, -3, [1, 5, 0, 1]
    elif case == 'ended twice':                     # more pages come back than there are
        lengths, table, new, n_free = [48, 48, 48, 48], [[0, 1, 2]] * 4, [-1, -1, -1, -1], 0
    else:
        new = [2 ** 31 - 1, 2 ** 31 - 1, 0, 1]
    for size in (dict(T=40), dict(R=32)):
        want = plan_oracle(lengths, new, table, free, n_free, page, **size)
        got = run_plan(lengths, new, table, free, n_free, page, **size)
        assert got == want


@pytest.mark.parametrize('B,T', [(3, 40000), (300, 200000)])
def test_page_plan_of_long_packed_prompts(B, T):
    page = 32
    g = torch.Generator().manual_seed(T)
    cuts = torch.sort(torch.randint(0, T - 99, (B - 1,), generator=g)).values.tolist()
    new = [b - a for a, b in zip([0] + cuts, cuts + [T - 99])]
    P = -(-max(new) // page) + 1
    n = sum(-(-x // page) for x in new) + 5
    lengths, table, free = [0] * B, [[-1] * P for _ in range(B)], torch.randperm(n, generator=g).tolist()
    want = plan_oracle(lengths, new, table, free, n, page, T=T)
    for in_place in (False, True):
        assert run_plan(lengths, new, table, free, n, page, T=T, in_place=in_place) == want


@pytest.mark.parametrize('B,longest,ends,size', [(300, 3000, lambda b: b % 3 == 1, dict(R=1)), (64, 5000, lambda b: b % 2 == 0, dict(T=1500)),
                                                 (1200, 160, lambda b: b % 7 != 0, dict(R=2)), (1000, 50000, lambda b: b in (3, 400, 401, 999), dict(T=1000)),
                                                 (2, 99999, lambda b: b == 0, dict(R=1000)), (5000, 100, lambda b: b % 2 == 1, dict(T=4000))])
@pytest.mark.parametrize('twice', [False, True])
def test_page_plan_takes_back_many_pages(B, longest, ends, size, twice):
    """More pages come back than the one workgroup has threads; twice: as many again as there are, where it has to stop."""
    page, g = 16, torch.Generator().manual_seed(B)
    lengths = [int(torch.randint(0, longest + 1 if ends(b) else 41, (1,), generator=g)) for b in range(B)]
    P = -(-longest // page) + 1
    used = [-(-n // page) for n in lengths]
    n = sum(used) + 3
    ids, table, at = torch.randperm(n, generator=g).tolist(), [], 0
    for u in used:
        table.append(ids[at:at + u] + [-5] * (P - u))
        at += u
    back = sum(u for b, u in enumerate(used) if ends(b))
    assert back > 4096
    free, n_free = ids[at:] + [-9] * at, n - at
    if twice:
        n_free = n - back // 2                       # (some of what is on the stack is held as well)
        free = (ids[::-1])[:n_free] + [-9] * (n - n_free)
    new = [-1 if ends(b) else b % 3 for b in range(B)]
    want = plan_oracle(lengths, new, table, free, n_free, page, **size)
    assert run_plan(lengths, new, table, free, n_free, page, **size) == want


def test_page_plan_keeps_every_page_exactly_once():
    """A serving loop with requests that come, grow, wait and end: no page is lost or held twice, in place over many steps."""
    B, P, page, n = 70, 6, 16, 150
    g = torch.Generator().manual_seed(5)
    lengths, table, free, n_free = dev([0] * B), torch.full((B, P), -1, dtype=torch.int32, device=DEV), dev(list(range(n))), dev([n])
    slots, refused = torch.empty(B, 40, dtype=torch.int32, device=DEV), dev([0])
    turned_away = 0
    for _ in range(60):
        pick = torch.rand(B, generator=g)
        new = torch.where(pick < 0.06, -1, torch.where(pick < 0.2, 0, torch.where(pick < 0.3, 33, 1)))
        ops.page_plan(lengths, dev(new.tolist()), table, free, n_free, page, slots, refused=refused)
        turned_away += refused.item()
        held = []
        for row, length in zip(table.tolist(), lengths.tolist()):
            held += row[:-(-length // page)]
        assert sorted(held + free.tolist()[:n_free.item()]) == list(range(n))
        live = slots[slots >= 0].tolist()
        assert len(set(live)) == len(live)
    assert turned_away > 0


# ---------------------------------------------------------------------------------------------------------------- write
def cache_pair(n_pages, page, Hk, D, kind, order='head', seed=0):
    """Two caches in one of the two memory orders, with a value of its own at every place."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for _ in range(2):
        if order == 'head':
            c = torch.randn(n_pages, Hk, page, D, generator=g, device=DEV).to(kind)
        elif order == 'token':
            c = torch.randn(n_pages, page, Hk, D, generator=g, device=DEV).to(kind).transpose(1, 2)
        else:                                       # rows with a gap behind them, heads with a gap behind them
            c = torch.randn(n_pages, Hk + 1, page + 3, D + 16, generator=g, device=DEV).to(kind)[:, :Hk, :page, :D]
        out.append(c)
    return out


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('order', ['head', 'token', 'gaps'])
@pytest.mark.parametrize('T,Hk,D,page', [(1, 1, 32, 16), (33, 4, 64, 16), (130, 3, 128, 48), (7, 5, 40, 16), (999, 2, 96, 64)])
def test_page_write_is_exact(kind, order, T, Hk, D, page):
    g = torch.Generator().manual_seed(T + D)
    n_pages = T // page + 4
    rows = torch.randn(T, 3 * Hk * D + 4, generator=g) * torch.exp(4 * torch.randn(T, 1, generator=g))
    rows[0, :8] = torch.tensor([0.0, -0.0, float('inf'), -float('inf'), float('nan'), 1e-40, 70000.0, 65519.996])
    rows = rows.to(DEV)
    k, v = rows[:, Hk * D:2 * Hk * D], rows[:, 2 * Hk * D:3 * Hk * D]
    kc, vc = cache_pair(n_pages, page, Hk, D, TYPES[kind], order)
    slots = torch.randperm(n_pages * page, generator=g)[:T]
    slots[1::5] = -1
    if T > 10:
        slots[3], slots[8] = n_pages * page, 2 ** 31 - 1        # places outside the cache
    want = []
    for x, c in ((k, kc), (v, vc)):
        w = c.cpu().clone().contiguous()
        for t in range(T):
            s = int(slots[t])
            if 0 <= s < n_pages * page:
                w[s // page, :, s % page] = x[t].cpu().reshape(Hk, D).to(TYPES[kind])
        want.append(w)
    ops.page_write(k, v, kc, vc, slots.to(torch.int32).to(DEV))
    for c, w in zip((kc, vc), want):
        a, b = c.cpu().contiguous().float(), w.float()
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, nan=3.0), torch.nan_to_num(b, nan=3.0))


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('T,Hk,D,order', [(9000, 8, 64, 'head'), (4001, 12, 128, 'token'), (70000, 1, 72, 'gaps')])
def test_page_write_of_many_rows(kind, T, Hk, D, order):
    """Writes large enough for streaming stores, against one assignment."""
    page = 32
    n_pages = T // page + 9
    kc, vc = cache_pair(n_pages, page, Hk, D, TYPES[kind], order)
    g = torch.Generator(device=DEV).manual_seed(T)
    rows = torch.randn(T, 2 * Hk * D, generator=g, device=DEV)
    slots = torch.randperm(n_pages * page, generator=g, device=DEV)[:T]
    slots[5::17] = -1
    want = []
    for x, c in ((rows[:, :Hk * D], kc), (rows[:, Hk * D:], vc)):
        w = c.clone(memory_format=torch.contiguous_format).transpose(1, 2).reshape(-1, Hk, D)
        w[slots[slots >= 0]] = x[slots >= 0].reshape(-1, Hk, D).to(TYPES[kind])
        want.append(w.view(n_pages, page, Hk, D).transpose(1, 2))
    ops.page_write(rows[:, :Hk * D], rows[:, Hk * D:], kc, vc, slots.int())
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_page_write_leaves_gaps_alone():
    base = [torch.full((6, 3, 19, 80), 5.0, device=DEV) for _ in range(2)]
    kc, vc = (c[:, :2, :16, :64] for c in base)
    rows = torch.randn(96, 128, device=DEV)
    ops.page_write(rows, rows, kc, vc, torch.randperm(96, device=DEV).int())
    for c in base:
        outside = torch.ones_like(c, dtype=torch.bool)
        outside[:, :2, :16, :64] = False
        assert bool((c[outside] == 5.0).all()) and not bool((c[:, :2, :16, :64] == 5.0).any())


# ------------------------------------------------------------------------------------------------------------ attention
def attention_oracle(q, kc, vc, table, lengths, heads, mask, scale, max_len):
    """float64, on the CPU: (ctx, bound on the error)."""
    B, (n_pages, Hk, page, D) = len(lengths), kc.shape
    G = heads // Hk
    out, bound = torch.zeros(B, heads, D, dtype=torch.float64), torch.zeros(B, heads, D, dtype=torch.float64)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), table.shape[1] * page, max_len)
        pos = torch.arange(n)
        ids = table[b].long()[pos // page]
        keep = (ids >= 0) & (ids < n_pages)
        if mask is not None:
            keep &= mask[b, :n] == 0
        ids, off = ids[keep], pos[keep] % page
        if not len(ids):
            continue
        for h in range(Hk):
            k, v = kc[ids, h, off].double(), vc[ids, h, off].double()
            for x in range(h * G, (h + 1) * G):
                qx = q[b, x * D:(x + 1) * D].double()
                w = torch.softmax(k @ qx * scale, 0)
                out[b, x] = w @ v
                bound[b, x] = attention_bound(qx, k, v, w, scale)
    return out.view(B, -1), bound.view(B, -1)


def attention_bound(q, k, v, w, scale):
    """With u = 2^-24: a score is a sum of D products, each operand exact to 4u (the 16-bit kinds split a query into pieces that hold 22 bits
    or more), plus the rounding of scale log2(e) q and of the score: error at most (D + 12) u sum |q k| scale + 2 u |score| = e.
    A weight changes by a factor within 1 +- (2 e + 8u) against the common normalisation (its own error and the sum's, exp2 to 2 ulp);
    the split of a weight into pieces adds 4u, sums over n rows in any order n u each for numerator and denominator, the rescaling when
    a maximum moves 2 u a time and at most once per 16 rows."""
    u, n, D, scale = 2.0 ** -24, len(w), len(q), abs(scale)
    e = ((D + 12) * u * (k.abs() @ q.abs()) * scale + 2 * u * (k @ q).abs() * scale).max()
    return (2 * float(e) + (16 + 2 * n + n / 8) * u) * (w @ v.abs()) + 1e-30


def pages_for(lengths, page, g, P=None, spare=3):
    used = [-(-max(int(n), 0) // page) for n in lengths]
    P = max(max(used), 1) if P is None else P
    n_pages = sum(used) + spare
    ids = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((len(used), P), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = torch.tensor(ids[at:at + u], dtype=torch.int32)
        at += u
    return table, n_pages


def check_attention(lengths, heads, Hk, D, page, kind, mask=None, order='head', scale=None, max_len=None, spoil=None, seed=0, spread=1.0, P=None,
                    cache_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    B = len(lengths)
    table, n_pages = pages_for(lengths, page, g, P)
    kc, vc = cache_pair(n_pages, page, Hk, D, TYPES[kind], order, seed)
    if cache_scale != 1.0:
        most = torch.finfo(kc.dtype).max                  # (a normal value 3.3 times 2e4 would be an infinity in float16)
        kc, vc = ((c.float() * cache_scale).clamp(-most, most).to(c.dtype) for c in (kc, vc))
    q = (torch.randn(B, heads * D + 8, generator=g) * spread).to(DEV)[:, :heads * D]
    P = table.shape[1]
    if spoil is not None:
        spoil(table, kc, vc, mask)
    lens = torch.tensor(lengths, dtype=torch.int32)
    ctx = torch.full((B, heads * D + 16), 9.0, device=DEV)
    view = ctx[:, 8:8 + heads * D]
    ops.paged_attention(q, kc, vc, table.to(DEV), lens.to(DEV), view, heads, key_mask=None if mask is None else mask.to(DEV), scale=scale,
                        max_len=max_len)
    want, bound = attention_oracle(q.cpu(), kc.cpu(), vc.cpu(), table, lens, heads, mask, 1 / math.sqrt(D) if scale is None else scale,
                                   P * page if max_len is None else min(max_len, P * page))
    got = view.cpu().double()
    assert bool(torch.isfinite(got).all())
    off = (got - want).abs()
    assert bool((off <= bound).all()), (float((off / bound.clamp(min=1e-30)).max()), float(off.max()))
    assert bool((ctx[:, :8] == 9.0).all()) and bool((ctx[:, 8 + heads * D:] == 9.0).all())
    return got


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('D', [32, 64, 128])
@pytest.mark.parametrize('heads,Hk,page', [(4, 4, 16), (8, 2, 48), (3, 1, 32), (16, 1, 64), (24, 1, 16), (40, 2, 128)])
def test_attention_around_tiles_and_pages(kind, D, heads, Hk, page):
    check_attention([0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 127, 128, 129, 200], heads, Hk, D, page, kind, seed=D + heads)


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('heads,Hk,D,page,lengths', [(8, 2, 64, 16, [5000]), (4, 4, 64, 16, [1, 4097, 0, 700]), (32, 8, 128, 64, [3001, 77]),
                                                     (6, 2, 32, 256, [9000, 1, 2, 3, 2999]), (20, 1, 64, 48, [2500, 2500])])
def test_attention_over_long_requests(kind, heads, Hk, D, page, lengths):
    check_attention(lengths, heads, Hk, D, page, kind, seed=heads)


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('B', [65, 300])
def test_attention_of_many_requests(kind, B):
    g = torch.Generator().manual_seed(B)
    check_attention(torch.randint(0, 400, (B,), generator=g).tolist(), 4, 2, 32, 16, kind, seed=B)


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('B', [3, 257, 1000])
def test_attention_of_many_requests_beside_long_ones(kind, B):
    """The line of all rows cut into parts: many requests to a part, several parts to a request, requests without rows."""
    g = torch.Generator().manual_seed(B)
    lengths = torch.randint(0, 90, (B,), generator=g).tolist()
    lengths[B // 2], lengths[0], lengths[-1] = 2600, 1100, 0
    check_attention(lengths, 4, 2, 64, 16, kind, seed=B)


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('D', [32, 64, 128])
@pytest.mark.parametrize('heads,Hk', [(4, 4), (8, 4), (24, 4), (80, 4)])
@pytest.mark.parametrize('masked', [False, True])
def test_attention_when_the_rows_could_be_many(kind, D, heads, Hk, masked):
    """A bound on the lengths of more than 100 MB of rows: the kernels whose loads of V stream past the caches."""
    lengths = [0, 1, 16, 33, 100, 1300, 517, 64]
    P = 32768 // 16 if D * (4 if kind == 'f32' else 2) < 256 else 16384 // 16
    assert 2 * len(lengths) * P * 16 * Hk * D * (4 if kind == 'f32' else 2) > 100e6
    mask = None
    if masked:
        mask = (torch.rand(len(lengths), P * 16, generator=torch.Generator().manual_seed(D)) < 0.3).float()
        mask[3] = 1.0
    check_attention(lengths, heads, Hk, D, 16, kind, mask=mask, seed=D, P=P)


@pytest.mark.parametrize('kind,cache_scale', [('f16', 1e-6), ('f16', 2e4), ('bf16', 1e-30), ('bf16', 1e30), ('f32', 1e-30), ('f32', 1e30)])
@pytest.mark.parametrize('heads', [2, 6])
def test_attention_over_the_range_of_the_cache_types(kind, cache_scale, heads):
    """float16 subnormals and values near its end; scores kept moderate by the scale."""
    check_attention([90, 1400], heads, 2, 64, 16, kind, scale=0.1 / cache_scale if cache_scale < 1e20 else 1e-31, cache_scale=cache_scale, seed=12)


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('order', ['token', 'gaps'])
def test_attention_with_other_strides(kind, order):
    check_attention([100, 37, 1600], 6, 3, 64, 32, kind, order=order, seed=3)


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('long', [False, True])
def test_attention_with_masks(kind, long):
    """Masks with any value but 0 leave rows out (NaN, infinities, the lowest value), some requests keep one row, some none."""
    lengths = [70, 1, 64, 33, 2000 if long else 90, 130, 48]
    g = torch.Generator().manual_seed(1)
    P = -(-max(lengths) // 16)
    mask = (torch.rand(len(lengths), P * 16, generator=g) < 0.4).float()
    mask[mask != 0] = torch.tensor([1.0, -1.0, float('nan'), float('inf'), -float('inf'), torch.finfo(torch.float32).min])[torch.randint(
        0, 6, (int((mask != 0).sum()),), generator=g)]
    mask[1], mask[2] = 1.0, 1.0                     # nothing left
    mask[3] = 1.0
    mask[3, 32] = 0.0                               # one row left, the last
    mask[5] = 0.0
    mask[5, :128] = 1.0                             # whole tiles masked in front
    got = check_attention(lengths, 4, 2, 64, 16, kind, mask=mask, seed=2)
    assert bool((got[1] == 0).all()) and bool((got[2] == 0).all())


@pytest.mark.parametrize('kind', sorted(TYPES))
def test_attention_ignores_what_lies_in_masked_rows_and_behind_the_length(kind):
    lengths = [70, 33, 1000, 16]
    mask = torch.zeros(4, 63 * 16)
    mask[:, 5::7] = 1.0
    mask[2, 100:300] = 1.0
    state = {}

    def spoil(table, kc, vc, m):
        state['table'] = table.clone()
        for c, bad in ((kc, float('nan')), (vc, float('inf'))):
            for b, n in enumerate(lengths):
                for pos in range(-(-n // 16) * 16):
                    if pos >= n or m[b, pos] != 0:
                        c[int(table[b, pos // 16]), :, pos % 16] = bad if pos % 2 else float('nan')
    check_attention(lengths, 4, 4, 64, 16, kind, mask=mask, spoil=spoil, seed=8)


@pytest.mark.parametrize('kind', sorted(TYPES))
def test_attention_leaves_out_pages_that_do_not_exist(kind):
    def spoil(table, kc, vc, m):
        table[0, 1], table[2, 0], table[2, 3], table[3, :] = -1, kc.shape[0], 2 ** 31 - 1, -2 ** 31
    got = check_attention([100, 20, 600, 64], 4, 2, 32, 16, kind, spoil=spoil, seed=4)
    assert bool((got[3] == 0).all())


@pytest.mark.parametrize('kind', sorted(TYPES))
def test_attention_lengths_count_as_the_nearest_bound(kind):
    check_attention([-3, 50, 96], 2, 2, 64, 16, kind, seed=5)
    g = torch.Generator().manual_seed(6)
    kc, vc = cache_pair(8, 16, 2, 64, TYPES[kind])
    table = torch.arange(6, dtype=torch.int32).view(2, 3)
    q = torch.randn(2, 128, generator=g).to(DEV)
    outs = []
    for lens in ([48, 48], [2 ** 31 - 1, 49]):
        ctx = torch.empty(2, 128, device=DEV)
        outs.append(ops.paged_attention(q, kc, vc, table.to(DEV), dev(lens), ctx, 2))
    assert torch.equal(*outs)


@pytest.mark.parametrize('max_len', [1, 31, 64, 100, 5000])
def test_attention_max_len(max_len):
    check_attention([10, 64, 150], 4, 4, 64, 16, 'bf16', max_len=max_len, seed=7)


@pytest.mark.parametrize('kind', sorted(TYPES))
@pytest.mark.parametrize('scale,spread', [(0.0, 1.0), (-0.3, 1.0), (1.0, 6.0), (0.125, 1e-6), (0.125, 1e-30), (2e-5, 3e4)])
def test_attention_scales(kind, scale, spread):
    check_attention([90, 700], 4, 2, 64, 16, kind, scale=scale, spread=spread, seed=9)


@pytest.mark.parametrize('kind', ['f32', 'f16'])
def test_attention_with_cache_offsets_past_32_bits(kind):
    """Page ids whose element offsets pass 2^32."""
    Hk, D, page = 4, 128, 64
    n_pages = (1 << 32) // (Hk * D * page) + 40
    kc, vc = (torch.empty(n_pages, Hk, page, D, dtype=TYPES[kind], device=DEV) for _ in range(2))
    ids = [n_pages - 1, 3, n_pages - 30, n_pages // 2 + 1, n_pages - 2, 7]
    g = torch.Generator(device=DEV).manual_seed(0)
    rows = torch.randn(6 * page, Hk * D, generator=g, device=DEV)
    slots = torch.cat([torch.arange(i * page, (i + 1) * page) for i in ids]).int().to(DEV)
    ops.page_write(rows, -rows, kc, vc, slots)
    q = torch.randn(2, 8 * D, generator=g, device=DEV)
    table, lens = torch.tensor(ids, dtype=torch.int32).view(2, 3), [150, 192]
    ctx = torch.empty(2, 8 * D, device=DEV)
    ops.paged_attention(q, kc, vc, table.to(DEV), dev(lens), ctx, 8)
    # the same pages in a small cache
    small = [c[torch.tensor(ids, device=DEV)].contiguous() for c in (kc, vc)]
    assert torch.equal(small[0].transpose(1, 2).reshape(-1, Hk * D), rows.to(TYPES[kind]))
    again = torch.empty_like(ctx)
    ops.paged_attention(q, *small, torch.arange(6, dtype=torch.int32).view(2, 3).to(DEV), dev(lens), again, 8)
    assert torch.equal(ctx, again)
    want, bound = attention_oracle(q.cpu(), small[0].cpu(), small[1].cpu(), torch.arange(6).view(2, 3), lens, 8, None, 1 / math.sqrt(D), 192)
    assert bool(((ctx.cpu().double() - want).abs() <= bound).all())


def test_attention_is_the_same_every_time_and_beside_others():
    """Two streams at once, each with calls of its own, against one at a time."""
    g = torch.Generator().manual_seed(11)
    lens = [3000, 17, 1200, 900]
    table, n_pages = pages_for(lens, 32, g)
    kc, vc = cache_pair(n_pages, 32, 4, 64, torch.bfloat16)
    qs = [torch.randn(4, 8 * 64, generator=g).to(DEV) for _ in range(12)]
    args = (kc, vc, table.to(DEV), dev(lens))
    alone = [ops.paged_attention(q, *args, torch.empty(4, 512, device=DEV), 8) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty(4, 512, device=DEV) for _ in qs]
    torch.cuda.synchronize()
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            ops.paged_attention(q, *args, outs[i], 8)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))


# ---------------------------------------------------------------------------------------------------- a decoding loop
class Loop:
    """Plan, write and attention of a batch over several steps, as a decoder uses them."""

    def __init__(self, kind, B=5, H=4, Hk=2, D=64, page=16, P=8, n_pages=22):
        self.H, self.Hk, self.D, self.page, self.B = H, Hk, D, page, B
        self.kc, self.vc = ops.new_paged_cache(n_pages, page, Hk, D, dtype=TYPES[kind], device=DEV)
        self.lengths, self.new = dev([0] * B), dev([0] * B)
        self.table = torch.full((B, P), -1, dtype=torch.int32, device=DEV)
        self.free, self.n_free = dev(list(range(n_pages))), dev([n_pages])
        self.slots = torch.empty(B, 1, dtype=torch.int32, device=DEV)
        self.qkv, self.ctx = torch.zeros(B, (H + 2 * Hk) * D, device=DEV), torch.zeros(B, H * D, device=DEV)

    def step(self):
        H, Hk, D = self.H, self.Hk, self.D
        ops.page_plan(self.lengths, self.new, self.table, self.free, self.n_free, self.page, self.slots)
        ops.page_write(self.qkv[:, H * D:(H + Hk) * D], self.qkv[:, (H + Hk) * D:], self.kc, self.vc, self.slots)
        ops.paged_attention(self.qkv[:, :H * D], self.kc, self.vc, self.table, self.lengths, self.ctx, H)


def feeds(B, width, steps, seed):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i in range(steps):
        pick = torch.rand(B, generator=g)
        new = torch.where(pick < 0.08, -1, torch.where(pick < 0.15, 0, 1)) if i > 3 else torch.ones(B)
        out.append((torch.randn(B, width, generator=g), new.int()))
    return out


@pytest.mark.parametrize('kind', sorted(TYPES))
def test_a_decoding_loop_matches_dense_histories(kind):
    loop = Loop(kind)
    H, Hk, D, B = loop.H, loop.Hk, loop.D, loop.B
    seen = [([], []) for _ in range(B)]
    for rows, new in feeds(B, (H + 2 * Hk) * D, 90, 3):
        loop.qkv.copy_(rows)
        loop.new.copy_(new)
        before = loop.lengths.tolist()
        loop.step()
        after = loop.lengths.tolist()
        ctx = loop.ctx.cpu().double()
        for b in range(B):
            if new[b] < 0:
                seen[b] = ([], [])
            elif after[b] == before[b] + 1:
                for x, at in zip(seen[b], (H, H + Hk)):
                    x.append(rows[b, at * D:(at + Hk) * D].to(TYPES[kind]).double().view(Hk, D))
            assert len(seen[b][0]) == after[b]
            if not seen[b][0]:
                assert bool((ctx[b] == 0).all())
                continue
            k, v = (torch.stack(x, 1) for x in seen[b])                      # [Hk, n, D]
            for h in range(H):
                q = rows[b, h * D:(h + 1) * D].double()
                w = torch.softmax(k[h * Hk // H] @ q / math.sqrt(D), 0)
                want = w @ v[h * Hk // H]
                off = (ctx[b, h * D:(h + 1) * D] - want).abs()
                assert bool((off <= attention_bound(q, k[h * Hk // H], v[h * Hk // H], w, 1 / math.sqrt(D))).all())


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
def test_a_captured_step_plans_writes_and_attends_on_every_replay(kind):
    eager, held = Loop(kind), Loop(kind)
    plan = feeds(eager.B, eager.qkv.shape[1], 60, 4)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        held.step()                                 # (new is zero: nothing changes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.step()
    for rows, new in plan:
        for loop in (eager, held):
            loop.qkv.copy_(rows)
            loop.new.copy_(new)
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for name in ('ctx', 'lengths', 'table', 'free', 'n_free', 'slots', 'kc', 'vc'):
            assert torch.equal(getattr(eager, name), getattr(held, name)), name


def test_two_captured_steps_replay_side_by_side():
    """Two graphs with loops of their own, replayed at once on two streams: they share no scratch."""
    loops = [Loop('bf16', B=3, P=130, n_pages=400) for _ in range(4)]            # two captured, two eager
    graphs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for i, loop in enumerate(loops):                # a long prompt each, so that the attention is split
        n = 1900 + 50 * (i % 2)
        g = torch.Generator().manual_seed(i % 2)
        rows = torch.randn(3 * n, 2 * loop.Hk * loop.D, generator=g).to(DEV)
        slots = torch.empty(3, n, dtype=torch.int32, device=DEV)
        ops.page_plan(loop.lengths, dev([n, n, n]), loop.table, loop.free, loop.n_free, loop.page, slots)
        ops.page_write(rows[:, :loop.Hk * loop.D], rows[:, loop.Hk * loop.D:], loop.kc, loop.vc, slots)
    torch.cuda.synchronize()
    for loop, s in zip(loops, streams):
        with torch.cuda.stream(s):
            loop.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loop.step()
        graphs.append(graph)
    for step in range(12):
        for i, loop in enumerate(loops):
            g = torch.Generator().manual_seed(100 + 2 * step + i % 2)
            loop.qkv.copy_(torch.randn(*loop.qkv.shape, generator=g))
            loop.new.fill_(1)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for loop in loops[2:]:
            loop.step()
        torch.cuda.synchronize()
        for a, b in zip(loops[:2], loops[2:]):
            assert torch.equal(a.ctx, b.ctx) and torch.equal(a.lengths, b.lengths) and torch.equal(a.kc, b.kc)


def test_a_step_program_issues_the_three_operators():
    """Plan, write and attention recorded into a step program, against the same calls one by one."""
    one, other = Loop('f32'), Loop('f32')
    steps = 20
    g = torch.Generator().manual_seed(2)
    rows = torch.randn(steps, one.B, one.qkv.shape[1], generator=g).to(DEV)
    outs = torch.zeros(2, steps, one.B, one.ctx.shape[1], device=DEV)

    def record(loop, out):
        H, Hk, D = loop.H, loop.Hk, loop.D

        def step(i):
            x = rows[i]
            ops.page_plan(loop.lengths, loop.new, loop.table, loop.free, loop.n_free, loop.page, loop.slots)
            ops.page_write(x[:, H * D:(H + Hk) * D], x[:, (H + Hk) * D:], loop.kc, loop.vc, loop.slots)
            ops.paged_attention(x[:, :H * D], loop.kc, loop.vc, loop.table, loop.lengths, out[i], H)
        return step

    for loop in (one, other):
        loop.new.fill_(1)
    program = ops.StepProgram(record(one, outs[0]))
    direct = record(other, outs[1])
    for i in range(steps):
        program.run(i)
        direct(i)
    assert torch.equal(outs[0], outs[1]) and bool((outs[0].abs().sum(-1) > 0).all())
    assert one.lengths.tolist() == [steps] * one.B


# -------------------------------------------------------------------------------------------------- the two ways to issue a call
def python_path(monkeypatch):
    monkeypatch.setattr(ops, '_issue', lambda: None)


@pytest.mark.parametrize('kind', sorted(TYPES))
def test_the_c_module_and_the_python_path_issue_the_same_launches(monkeypatch, kind):
    """A loop through csrc/hostops.cpp and one through the Python path: the same bits everywhere.  While the first runs the argument blocks of
    the second are out of reach, so that it cannot have taken that path."""
    width, steps = Loop(kind).qkv.shape[1], 24
    plan = feeds(5, width, steps, 21)
    blocks = {n: getattr(ops._lib, n) for n in ('PagePlanArgs', 'PageWriteArgs', 'PagedAttentionArgs')}
    loops = []
    for fast in (True, False):
        with monkeypatch.context() as mp:
            if fast:
                for n in blocks:
                    mp.setattr(ops._lib, n, None)
            else:
                python_path(mp)
            loop = Loop(kind, P=130, n_pages=700)
            big = torch.randn(5 * 1300, 2 * loop.Hk * loop.D, generator=torch.Generator().manual_seed(1)).to(DEV)
            slots, positions, refused = (torch.empty(s, dtype=torch.int32, device=DEV) for s in ((6513,), (6513,), (1,)))
            ops.page_plan(loop.lengths, dev([1300, 700, 0, 1300, 1200]), loop.table, loop.free, loop.n_free, loop.page, slots, positions=positions,
                          refused=refused)
            ops.page_write(big[:, :loop.Hk * loop.D], big[:, loop.Hk * loop.D:], loop.kc, loop.vc, slots[:6500])
            seen = []
            for rows, new in plan:
                loop.qkv.copy_(rows)
                loop.new.copy_(new)
                loop.step()
                masked = ops.paged_attention(loop.qkv[:, :loop.H * loop.D], loop.kc, loop.vc, loop.table, loop.lengths, torch.zeros_like(loop.ctx), loop.H,
                                             key_mask=(torch.arange(2080, device=DEV) % 3 == 1).float().expand(5, 2080), scale=0.2, max_len=1900)
                seen += [loop.ctx.clone(), masked, loop.lengths.clone(), loop.slots.clone()]
            loops.append(seen + [slots, positions, refused, loop.table, loop.free, loop.n_free, loop.kc, loop.vc])
    assert all(torch.equal(a, b) for a, b in zip(*loops)) and len(loops[0]) == len(loops[1])


def good_calls():
    g = torch.Generator().manual_seed(3)
    kc, vc = cache_pair(12, 16, 2, 64, torch.float32)
    kc16, _ = cache_pair(12, 16, 2, 64, torch.float16)
    q, rows = torch.randn(3, 256, generator=g).to(DEV), torch.randn(3, 128, generator=g).to(DEV)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
    attend = dict(q=q, k_cache=kc, v_cache=vc, block_table=i32(3, 4), lengths=i32(3), ctx=torch.zeros(3, 256, device=DEV), heads=4)
    write = dict(k=rows, v=rows, k_cache=kc, v_cache=vc, slots=i32(3))
    plan = dict(lengths=i32(3), new=i32(3), block_table=i32(3, 4), free_pages=i32(12), n_free=i32(1), page=16, slots=i32(3, 1))
    f = lambda *s: torch.zeros(*s, device=DEV)
    bad = [(ops.paged_attention, attend, b) for b in (
        dict(q=q.half()), dict(q=q[:, :255]), dict(q=q.t()), dict(q=q.cpu()), dict(ctx=f(2, 256)), dict(ctx=f(3, 256).cpu()), dict(heads=3), dict(heads=0),
        dict(k_cache=kc16), dict(k_cache=kc16.double(), v_cache=kc16.double()), dict(k_cache=kc[:, :, :, ::2], v_cache=vc[:, :, :, ::2]),
        dict(v_cache=vc[:5]), dict(block_table=i32(4, 4)), dict(block_table=i32(4, 3).t()), dict(block_table=i32(3, 4).long()), dict(lengths=i32(3).long()),
        dict(lengths=i32(6)[::2]), dict(key_mask=f(3, 63)), dict(key_mask=f(3, 64).bool()), dict(key_mask=f(3, 64).cpu()), dict(max_len=0), dict(max_len=-5),
        dict(k_cache=kc[:, :, :8], v_cache=vc[:, :, :8]), dict(q=f(3, 257)[:, 1:]))]
    bad += [(ops.page_write, write, b) for b in (
        dict(k=rows[:2]), dict(v=rows[:, :100]), dict(k=rows.half()), dict(slots=i32(4)), dict(slots=i32(3).long()), dict(slots=i32(6)[::2]), dict(slots=i32(3).cpu()),
        dict(k_cache=kc[:1].expand(12, 2, 16, 64), v_cache=vc[:1].expand(12, 2, 16, 64)), dict(k_cache=kc16), dict(k=f(3, 129)[:, 1:]), dict(k_cache=kc[:, :, :5], v_cache=vc[:, :, :5]))]
    bad += [(ops.page_plan, plan, b) for b in (
        dict(new=i32(4)), dict(new=i32(3).long()), dict(block_table=i32(2, 4)), dict(free_pages=i32(12).cpu()), dict(n_free=i32(2)), dict(page=8), dict(page=-16),
        dict(slots=i32(2, 1)), dict(slots=i32(3, 2)[:, :1]), dict(slots=i32(1, 3, 1)), dict(positions=i32(3)), dict(lengths_out=i32(4)), dict(n_free_out=i32(3)),
        dict(refused=f(1)), dict(lengths=i32(3).cpu()))]
    return bad


@pytest.mark.parametrize('python', [False, True])
def test_both_ways_refuse_the_same_calls(monkeypatch, python):
    if python:
        python_path(monkeypatch)
    for fn, good, bad in good_calls():
        fn(**good)
        with pytest.raises((ValueError, TypeError, ops._lib.EsttsError)):
            fn(**dict(good, **bad))
            raise AssertionError(f'{fn.__name__} took {[(k, getattr(v, "shape", v)) for k, v in bad.items()]}')


def test_calls_the_c_module_leaves_to_python_work(monkeypatch):
    """Sizes and scales that are not plain Python numbers, one-row views with any stride, caches with dimensions of one."""
    kc, vc = cache_pair(1, 16, 1, 64, torch.float32)
    q = torch.randn(1, 300, device=DEV)[:, :64]
    args = (kc, vc, torch.zeros(1, 1, dtype=torch.int32, device=DEV), dev([9]))
    a = ops.paged_attention(q, *args, torch.empty(1, 64, device=DEV), 1, scale=1, max_len=16)
    b = ops.paged_attention(q, *args, torch.empty(1, 64, device=DEV), 1, scale=1.0, max_len=16.0)
    python_path(monkeypatch)
    assert torch.equal(a, b) and torch.equal(a, ops.paged_attention(q, *args, torch.empty(1, 64, device=DEV), 1, scale=1.0))


class Named(torch.Tensor):
    pass


def test_parameters_subclasses_and_large_offsets_are_taken_by_either_path():
    kc, vc = cache_pair(40, 16, 2, 64, torch.float16)
    g = torch.Generator().manual_seed(4)
    for c in (kc, vc):
        c.copy_(torch.randn(c.shape, generator=g))
    q = torch.randn(2, 256, generator=g).to(DEV)
    args = (kc, vc, torch.arange(40, dtype=torch.int32, device=DEV).view(2, 20), dev([300, 77]))
    attend = lambda x, *a: ops.paged_attention(x, *(a or args), torch.empty(2, 256, device=DEV), 4)
    want = attend(q)
    assert torch.equal(want, attend(torch.nn.Parameter(q))) and torch.equal(want, attend(q.as_subclass(Named)))
    assert torch.equal(want, attend(q, kc.as_subclass(Named), *args[1:]))


def test_scratch_goes_back_to_the_allocator():
    """Calls in two launches, good and bad ones, on two streams: what is allocated afterwards is what was before."""
    kc, vc = cache_pair(600, 16, 2, 64, torch.bfloat16)
    q, ctx = torch.randn(3, 256, device=DEV), torch.empty(3, 256, device=DEV)
    table, lengths = torch.arange(600, dtype=torch.int32, device=DEV).view(3, 200), dev([3200, 1, 1700])
    slots, free, n_free, new = (torch.empty(6000, dtype=torch.int32, device=DEV), torch.arange(600, dtype=torch.int32, device=DEV), dev([0]), dev([0, 0, 0]))
    assert ops._lib.load().estts_paged_attention_ws_bytes(3, 4, 2, 64, 3200, 1) > 0 and ops._lib.load().estts_page_plan_ws_bytes(3, 6000) > 0
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            for _ in range(20):
                ops.paged_attention(q, kc, vc, table, lengths, ctx, 4)
                ops.page_plan(lengths, new, table, free, n_free, 16, slots)
                with pytest.raises(ops._lib.EsttsError):
                    ops.page_plan(lengths, new, table, free, n_free, 24, slots)
        torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


# ------------------------------------------------------------------- the same conditions for every kernel: one, two, three queries a key head; cut or not
EVERY_KERNEL = [pytest.mark.parametrize('kind', sorted(TYPES)), pytest.mark.parametrize('group', [1, 2, 3]), pytest.mark.parametrize('long', [False, True])]


def every_kernel(test):
    for mark in EVERY_KERNEL:
        test = mark(test)
    return test


@every_kernel
@pytest.mark.parametrize('D', [32, 128])
def test_every_kernel_ignores_what_lies_in_masked_rows_and_behind_the_length(kind, group, long, D):
    lengths = [70, 33, 2100 if long else 900, 16, 0, 129]
    mask = torch.zeros(6, -(-max(lengths) // 16) * 16)
    mask[:, 5::7] = 1.0
    mask[2, 100:300] = float('nan')
    mask[3] = torch.finfo(torch.float32).min          # nothing left

    def spoil(table, kc, vc, m):
        for c, bad in ((kc, float('inf')), (vc, float('nan'))):
            for b, n in enumerate(lengths):
                for pos in range(-(-n // 16) * 16):
                    if pos >= n or m[b, pos] != 0:
                        c[int(table[b, pos // 16]), :, pos % 16] = bad if pos % 2 else -float('inf')
    got = check_attention(lengths, 2 * group, 2, D, 16, kind, mask=mask, spoil=spoil, seed=8)
    assert bool((got[3:5] == 0).all())


@every_kernel
def test_every_kernel_leaves_out_pages_that_do_not_exist(kind, group, long):
    def spoil(table, kc, vc, m):
        table[0, 1], table[2, 0], table[2, 3], table[3, :] = -1, kc.shape[0], 2 ** 31 - 1, -2 ** 31
    got = check_attention([100, 20, 2050 if long else 600, 64], 2 * group, 2, 64, 16, kind, spoil=spoil, seed=4)
    assert bool((got[3] == 0).all())


@every_kernel
@pytest.mark.parametrize('order', ['token', 'gaps'])
def test_every_kernel_takes_other_strides(kind, group, long, order):
    check_attention([100, 37, 1600 if long else 400], 3 * group, 3, 64, 48, kind, order=order, seed=3)


@every_kernel
@pytest.mark.parametrize('scale,spread', [(-0.3, 1.0), (0.125, 1e-30), (2e-5, 3e4)])
def test_every_kernel_takes_other_scales(kind, group, long, scale, spread):
    check_attention([90, 1700 if long else 700], 2 * group, 2, 64, 16, kind, scale=scale, spread=spread, seed=9)


@pytest.mark.parametrize('kind', ['bf16', 'f32'])
@pytest.mark.parametrize('heads', [4, 16])
def test_every_kernel_reaches_cache_offsets_past_32_bits(kind, heads):
    Hk, D, page = 4, 128, 64
    n_pages = (1 << 32) // (Hk * D * page) + 40
    kc, vc = (torch.empty(n_pages, Hk, page, D, dtype=TYPES[kind], device=DEV) for _ in range(2))
    ids = [n_pages - 1, 3, n_pages - 30, n_pages // 2 + 1, n_pages - 2, 7]
    g = torch.Generator(device=DEV).manual_seed(1)
    rows = torch.randn(6 * page, Hk * D, generator=g, device=DEV)
    ops.page_write(rows, rows.flip(0), kc, vc, torch.cat([torch.arange(i * page, (i + 1) * page) for i in ids]).int().to(DEV))
    q = torch.randn(2, heads * D, generator=g, device=DEV)
    small = [c[torch.tensor(ids, device=DEV)].contiguous() for c in (kc, vc)]
    outs = [ops.paged_attention(q, *c, torch.tensor(t, dtype=torch.int32).view(2, 3).to(DEV), dev([150, 192]), torch.empty_like(q), heads)
            for c, t in (((kc, vc), ids), (small, list(range(6))))]
    want, bound = attention_oracle(q.cpu(), small[0].cpu(), small[1].cpu(), torch.arange(6).view(2, 3), [150, 192], heads, None, 1 / math.sqrt(D), 192)
    assert torch.equal(*outs) and bool(((outs[0].cpu().double() - want).abs() <= bound).all())


# ------------------------------------------------------------------------------------------------------- launches that fail
def test_a_launch_that_fails_is_issued_once_and_said(monkeypatch):
    """The C++ module's entry points answer -2 (an error of the runtime, the launch possibly under way): the call raises, and is not issued
    again by the Python path, which would plan the same rows twice.  -1 (refused, nothing issued) goes to the Python path as ever."""
    lib, calls, answer = ops._lib, [], [-2]
    entry = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)
    names = ('estts_page_plan', 'estts_page_write', 'estts_paged_attention')

    def said(name):
        def f(args, stream):
            calls.append(name)
            return answer[0]
        return entry(f)
    fakes = {n: said(n) for n in names}
    loop = Loop('f32')
    loop.new.fill_(1)
    H, Hk, D = loop.H, loop.Hk, loop.D
    k, v = loop.qkv[:, H * D:(H + Hk) * D], loop.qkv[:, (H + Hk) * D:]
    plan = lambda: ops.page_plan(loop.lengths, loop.new, loop.table, loop.free, loop.n_free, loop.page, loop.slots)
    write = lambda: ops.page_write(k, v, loop.kc, loop.vc, loop.slots)
    attend = lambda: ops.paged_attention(loop.qkv[:, :H * D], loop.kc, loop.vc, loop.table, loop.lengths, loop.ctx, H)
    plan()
    try:
        with monkeypatch.context() as mp:               # (only the C++ module's addresses: the Python path keeps the library's)
            for n in names:
                mp.setattr(lib.load(), n, fakes[n])
            lib._host = None
            lib.load_host()
        for call in (plan, write, attend):
            with pytest.raises(lib.EsttsError):
                call()
        assert calls == list(names) and loop.lengths.tolist() == [1] * loop.B
        answer[0] = -1
        plan()
        assert loop.lengths.tolist() == [2] * loop.B
    finally:
        lib._host = None
        lib.load_host()
    plan()
    assert loop.lengths.tolist() == [3] * loop.B and len(calls) == 4


# ------------------------------------------------------------------------------------------------ small values, bounded by themselves
@pytest.mark.parametrize('kind,scale_of', [('f16', 1e-6), ('f16', 2e4), ('bf16', 1e-30), ('bf16', 1e30), ('f32', 1e-30), ('f32', 1e30)])
@pytest.mark.parametrize('heads', [2, 4, 6])
@pytest.mark.parametrize('lengths', [[90, 700], [90, 1400]])
def test_attention_of_very_small_and_very_large_values(kind, scale_of, heads, lengths):
    """attention_bound without its absolute term, which is as large as outputs of 1e-30 are themselves.  In its place what can be lost where a
    product or a piece is below the smallest normal number: each of a row's at most three pieces and its product less than 2^-126, so
    (3 + 1) n 2^-126, 4e-35 at 700 rows where the outputs are some 4e-32.  Zeros in place of the outputs are out of these bounds."""
    g = torch.Generator().manual_seed(heads)
    table, n_pages = pages_for(lengths, 16, g)
    kc, vc = cache_pair(n_pages, 16, 2, 64, torch.float32, seed=5)
    most = torch.finfo(TYPES[kind]).max
    kc, vc = ((c * scale_of).clamp(-most, most).to(TYPES[kind]) for c in (kc, vc))
    q = torch.randn(2, heads * 64, generator=g)
    scale = 0.1 / scale_of if scale_of < 1e20 else 1e-31
    ctx = torch.full((2, heads * 64), 9.0, device=DEV)
    ops.paged_attention(q.to(DEV), kc, vc, table.to(DEV), dev(lengths), ctx, heads, scale=scale)
    want, bound = attention_oracle(q, kc.cpu(), vc.cpu(), table, lengths, heads, None, scale, table.shape[1] * 16)
    bound = (bound - 1e-30) + 4 * torch.tensor(lengths)[:, None] * 2.0 ** -126
    assert bool((want.abs().view(2, heads, 64).amax(-1) > 20 * bound.view(2, heads, 64).amax(-1)).all())
    assert bool(((ctx.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize('layout', ['packed', 'padded'])
def test_page_plan_where_requests_without_need_follow_refused_ones(layout):
    """The height of the stack goes down by the pages that were taken, not by what refused requests had asked for: requests that take a page, ask
    for more than there are, have room in their last page, end, have room, ask for more than there are."""
    lengths, new = [16, 16, 5, 40, 17, 16], [3, 40, 1, -1, 2, 200]
    table, free, n_free = [[0] + [-1] * 13, [1] + [-1] * 13, [2] + [-1] * 13, [3, 4, 5] + [-1] * 11, [6, 7] + [-1] * 12, [8] + [-1] * 13], list(range(9, 12)) + [-9] * 9, 3
    size = dict(T=300) if layout == 'packed' else dict(R=200)
    for stack in (3, 0):                             # (the one that ends gives three back)
        want = plan_oracle(lengths, new, table, free, stack, 16, **size)
        assert run_plan(lengths, new, table, free, stack, 16, **size) == want and want['n_free'] == 2
    got = run_plan([16, 16, 5], [3, 60, 1], table[:3], free, 3, 16, **(dict(T=64) if layout == 'packed' else dict(R=60)))
    assert got['n_free'] == 2 and got['refused'] == 1 and got['lengths'] == [19, 16, 6]

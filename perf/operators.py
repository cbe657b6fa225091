"""The operators of paged decoding as they are measured: the page plan, the write into the pages, the attention of one new token.

Several utterances decode side by side from one key / value memory that is cut into pages.  In every step the plan gives each
request the pages its new rows need and says where each row goes, the write puts the rows there, and each request's new row
attends everything the request has in its pages.  `own` False computes the operators in elementary torch operations, True
through the framework's entry points.
"""
import math

import torch

own = False
DEV = 'cuda'
TYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}


def listed():
    return [
        # every request of a serving batch advances by one row (what happens at each decoder step)
        dict(name='plan_step_32', op='plan', batch=32, page=16, longest=1000, prompt=0, ending=0, padded=True),
        # a batch of new requests whose prompts come packed one after another
        dict(name='plan_prompts_64', op='plan', batch=64, page=32, longest=0, prompt=2047, ending=0, padded=False),
        # a large batch in which requests end, advance and arrive at once, with too few pages for all
        dict(name='plan_churn_1000', op='plan', batch=1000, page=16, longest=4096, prompt=301, ending=7, padded=False),
        # the rows of one decoder step, decoder of four heads of 64, float32 pages
        dict(name='write_step_32', op='write', rows=32, kv_heads=4, depth=64, page=16, type='float32', holes=0),
        # the rows of packed prompts, some of them padding
        dict(name='write_prompts_bf16', op='write', rows=16411, kv_heads=8, depth=128, page=32, type='bfloat16', holes=9),
        # one utterance of a hundred positions in a decoder of four heads of 64: nothing but latency
        dict(name='attend_one_short', op='attend', batch=1, heads=4, kv_heads=4, depth=64, page=16, longest=100, ragged=False, mask=True, type='float32'),
        # a serving batch of that decoder with zero frames masked, and a request whose mask leaves nothing
        dict(name='attend_32_f32', op='attend', batch=32, heads=4, kv_heads=4, depth=64, page=16, longest=601, ragged=True, mask=True, type='float32'),
        # many requests of medium length with a key head for each query head, float32 pages
        dict(name='attend_200_f32', op='attend', batch=200, heads=8, kv_heads=8, depth=64, page=64, longest=1021, ragged=False, mask=False, type='float32'),
        # requests of very different lengths, four query heads to a key head
        dict(name='attend_ragged_bf16', op='attend', batch=61, heads=32, kv_heads=8, depth=128, page=32, longest=4096, ragged=True, mask=False, type='bfloat16'),
        # one very long request
        dict(name='attend_one_long', op='attend', batch=1, heads=32, kv_heads=8, depth=128, page=64, longest=131071, ragged=False, mask=False, type='bfloat16'),
        # all query heads on one key head, pages that are no power of two
        dict(name='attend_shared_f16', op='attend', batch=16, heads=16, kv_heads=1, depth=64, page=48, longest=8191, ragged=True, mask=False, type='float16'),
        # small heads, a few requests of a few thousand rows
        dict(name='attend_small_heads', op='attend', batch=3, heads=6, kv_heads=2, depth=32, page=128, longest=2500, ragged=True, mask=False, type='bfloat16'),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(['plan', 'write', 'attend', 'attend'])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    if op == 'plan':
        padded = rng.random() < 0.5
        return dict(op='plan', batch=_log(rng, 1, 1000), page=page, longest=_log(rng, 1, 4096), prompt=0 if padded else rng.choice([0, _log(rng, 2, 300)]),
                    ending=rng.choice([0, 3, 10]), padded=padded)
    kind, depth = rng.choice(list(TYPES)), rng.choice([32, 64, 128])
    if op == 'write':
        kv = rng.randint(1, 8)
        return dict(op='write', rows=_log(rng, 1, 16000 * 1024 // (kv * depth * 2)), kv_heads=kv, depth=depth, page=page, type=kind, holes=rng.choice([0, 2, 9]))
    kv, group = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 1, 2, 3, 4, 7, 8, 16, 24])
    batch = _log(rng, 1, 256)
    row = 2 * kv * depth * (4 if kind == 'float32' else 2)
    # (at most 0.3 GB of pages, and as much again as float32 scores in the plain form)
    most = min(60000, int(3e8 / (batch * row)), int(1.5e8 / (batch * kv * group)))
    return dict(op='attend', batch=batch, heads=kv * group, kv_heads=kv, depth=depth, page=page, longest=_log(rng, 1, max(1, most)),
                ragged=rng.random() < 0.6, mask=rng.random() < 0.3, type=kind)


# -------------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """How many rows each request has in its pages, in no order: a property of the case, so that every seed has the same work."""
    B, hi = case['batch'], case['longest']
    if case.get('ragged', True) and B > 1:
        return [max(1 if hi else 0, round(hi * (i + 1) / B)) for i in range(B)]
    return [hi] * B


def _shuffled(values, g):
    return torch.tensor(values, dtype=torch.int64)[torch.randperm(len(values), generator=g)]


def _news(case):
    """Rows that come for each request: -1 where it ends."""
    B, out = case['batch'], []
    for i in range(B):
        if case['ending'] and i % case['ending'] == 1:
            out.append(-1)
        elif case['prompt'] and (case['longest'] == 0 or i % 5 == 0):
            out.append(1 + (i * 37) % case['prompt'] if case['longest'] else max(1, round(case['prompt'] * (i + 1) / B)))
        else:
            out.append(0 if i % 11 == 3 else 1)
    return out


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=DEV).manual_seed(seed)
    page = case['page']

    def normal(*shape):
        return torch.randn(*shape, generator=gd, device=DEV)

    if case['op'] == 'plan':
        B = case['batch']
        length, new = _shuffled(_lengths(case), g), _shuffled(_news(case), g)
        used = (length + page - 1) // page
        want = new.clamp(min=0)
        P = (case['longest'] + int(want.max()) + page - 1) // page + 2
        need = (length + want + page - 1) // page - used
        # most of what is asked for is there, so that the last requests of a large batch are turned away
        n_free = int(need.sum()) if case['padded'] else max(1, int(need.sum()) * 9 // 10)
        n_pages = int(used.sum()) + B + int(want.sum()) // page                 # (some belong to nobody here)
        order = torch.randperm(n_pages, generator=g)
        first = torch.cumsum(used, 0) - used
        j = torch.arange(P)
        table = torch.where(j < used[:, None], order[(first[:, None] + j).clamp(max=n_pages - 1)], -1)
        free = torch.roll(order, -int(used.sum()))                              # what lies above the stack is of no meaning
        T = int(want.sum()) + (0 if case['padded'] else 13)
        i32 = dict(dtype=torch.int32, device=DEV)
        rows = torch.empty(B, 1, **i32) if case['padded'] else torch.empty(max(1, T), **i32)
        return dict(case=case, lengths=length.to(**i32), new=new.to(**i32), table=table.to(**i32), free=free.to(**i32),
                    n_free=torch.tensor([n_free], **i32), slots=rows, positions=torch.empty_like(rows), lengths_out=torch.empty(B, **i32),
                    n_free_out=torch.empty(1, **i32), refused=torch.empty(1, **i32))
    Hk, D, kind = case['kv_heads'], case['depth'], TYPES[case['type']]
    if case['op'] == 'write':
        T = case['rows']
        n_pages = (2 * T + page - 1) // page + 1
        slots = torch.randperm(n_pages * page, generator=g)[:T]
        if case['holes']:
            slots[torch.arange(T) % case['holes'] == 1] = -1
        rows = normal(T, 3 * Hk * D)                                            # q | k | v of the fused projection
        return dict(case=case, k=rows[:, Hk * D:2 * Hk * D], v=rows[:, 2 * Hk * D:], k_cache=normal(n_pages, Hk, page, D).to(kind),
                    v_cache=normal(n_pages, Hk, page, D).to(kind), slots=slots.to(dtype=torch.int32, device=DEV))
    B, H = case['batch'], case['heads']
    length = _shuffled(_lengths(case), g)
    used = (length + page - 1) // page
    n_pages = int(used.sum()) + 3
    order = torch.randperm(n_pages, generator=g)
    first = torch.cumsum(used, 0) - used
    P = int(used.max())
    j = torch.arange(P)
    table = torch.where(j < used[:, None], order[(first[:, None] + j).clamp(max=n_pages - 1)], -1)
    mask = None
    if case['mask']:
        mask = (torch.rand(B, P * page, generator=gd, device=DEV) < 0.1).float()
        if B > 1:
            mask[B // 2] = 1.0
    rows = normal(B, (H + 2 * Hk) * D)
    return dict(case=case, q=rows[:, :H * D], k_cache=normal(n_pages, Hk, page, D).to(kind), v_cache=normal(n_pages, Hk, page, D).to(kind),
                table=table.to(dtype=torch.int32, device=DEV), lengths=length.to(dtype=torch.int32, device=DEV), mask=mask, longest=case['longest'],
                ctx=torch.empty(B, H * D, device=DEV))


# --------------------------------------------------------------------------------------------------------------- plain forms
def _plan(s):
    page, P = s['case']['page'], s['table'].shape[1]
    length, new, table = s['lengths'].long(), s['new'].long(), s['table'].long()
    B, n_pages, dev = length.shape[0], s['free'].shape[0], length.device
    used, want, ends = (length + page - 1) // page, new.clamp(min=0), new < 0
    # the pages of the requests that end go onto the stack
    back = torch.where(ends, used, 0)
    at = s['n_free'].long() + torch.cumsum(back, 0) - back
    j = torch.arange(P, device=dev)
    free = torch.cat([s['free'].long(), s['free'].new_zeros(1).long()])
    free.scatter_(0, torch.where(ends[:, None] & (j < used[:, None]), at[:, None] + j, n_pages).view(-1), table.reshape(-1))
    free = free[:n_pages]
    top = s['n_free'].long() + back.sum()
    # first come, first served
    start = torch.cumsum(want, 0) - want
    padded = s['slots'].dim() == 2
    room = (want <= s['slots'].shape[1]) if padded else (start + want <= s['slots'].shape[0])
    fits = ~ends & room & (length + want <= P * page)
    need = torch.where(fits, (length + want + page - 1) // page - used, 0)
    upto = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (upto <= top))
    i = j - used[:, None]
    got = free[(top - 1 - (upto - need)[:, None] - i).clamp(0, n_pages - 1)]
    table = torch.where(granted[:, None] & (i >= 0) & (i < need[:, None]), got, table)
    # where each row goes
    if padded:
        b = torch.arange(B, device=dev)[:, None]
        i = torch.arange(s['slots'].shape[1], device=dev)[None]
        live = granted[:, None] & (i < want[:, None])
    else:
        t = torch.arange(s['slots'].shape[0], device=dev)
        b = torch.searchsorted(start + want, t, right=True)
        live = b < B
        b = b.clamp(max=B - 1)
        i = t - start[b]
        live = live & granted[b]
    pos = (length[b] + i).clamp(0, P * page - 1)
    slots = torch.where(live, table[b, pos // page] * page + pos % page, -1)
    i32 = torch.int32
    return dict(slots=slots.to(i32), positions=torch.where(live, length[b] + i, -1).to(i32), table=table.to(i32), free=free.to(i32),
                lengths=torch.where(ends, 0, torch.where(granted, length + want, length)).to(i32),
                n_free=(top - torch.where(granted, upto, 0).max()).to(i32), refused=(~ends & ~granted).sum().view(1).to(i32))


def _write(s):
    Hk, D, page = s['case']['kv_heads'], s['case']['depth'], s['case']['page']
    slot = s['slots'].long()
    out = []
    first = (slot >= 0).int().argmax()                                            # (rows without a place do what this one does)
    for rows, cache in ((s['k'], s['k_cache']), (s['v'], s['v_cache'])):
        value = rows.reshape(-1, Hk, D).to(cache.dtype)
        at = torch.where(slot < 0, slot[first], slot)
        cache[at // page, :, at % page] = torch.where((slot < 0)[:, None, None], value[first], value)
        out.append(cache)
    return dict(k_cache=out[0], v_cache=out[1])


def _attend(s):
    c = s['case']
    B, H, Hk, D, page, L = c['batch'], c['heads'], c['kv_heads'], c['depth'], c['page'], s['longest']
    pos = torch.arange(L, device=DEV)
    pages = s['table'].long()[:, pos // page].clamp(min=0)
    live = pos < s['lengths'][:, None]
    if s['mask'] is not None:
        live = live & (s['mask'][:, :L] == 0)
    k = s['k_cache'][pages, :, pos % page].float()                                # [B, L, Hk, D]
    v = torch.where(live[:, :, None, None], s['v_cache'][pages, :, pos % page].float(), 0.0)
    q = s['q'].reshape(B, Hk, H // Hk, D) * (1.0 / math.sqrt(D))
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous())                   # [B, Hk, G, L]
    score = torch.where(live[:, None, None], score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous()) / torch.where(total > 0, total, 1.0)
    return out.reshape(B, H * D)


def run(state):
    op = state['case']['op']
    if not own:
        return {'plan': _plan, 'write': _write, 'attend': _attend}[op](state)
    from estts import ops
    s = state
    if op == 'plan':
        ops.page_plan(s['lengths'], s['new'], s['table'], s['free'], s['n_free'], s['case']['page'], s['slots'], positions=s['positions'],
                      lengths_out=s['lengths_out'], n_free_out=s['n_free_out'], refused=s['refused'])
        return dict(slots=s['slots'], positions=s['positions'], table=s['table'], free=s['free'], lengths=s['lengths_out'],
                    n_free=s['n_free_out'], refused=s['refused'])
    if op == 'write':
        ops.page_write(s['k'], s['v'], s['k_cache'], s['v_cache'], s['slots'])
        return dict(k_cache=s['k_cache'], v_cache=s['v_cache'])
    return ops.paged_attention(s['q'], s['k_cache'], s['v_cache'], s['table'], s['lengths'], s['ctx'], s['case']['heads'], key_mask=s['mask'],
                               max_len=s['longest'])


def work(case):
    if case['op'] == 'plan':
        length, new, page = _lengths(case), _news(case), case['page']
        T = case['batch'] if case['padded'] else sum(max(n, 0) for n in new) + 13
        pages = sum(max(n, 0) for n in new) // page + sum(length) // page * sum(n < 0 for n in new) // len(new)
        return {'bytes': 4.0 * (3 * case['batch'] + 2 * pages + 2 * T), 'flops': 0.0}
    es = 4 if case['type'] == 'float32' else 2
    if case['op'] == 'write':
        live = case['rows'] - (case['rows'] // case['holes'] if case['holes'] else 0)
        return {'bytes': 2.0 * live * case['kv_heads'] * case['depth'] * (4 + es) + 4.0 * case['rows'], 'flops': 0.0}
    rows, B, H, D = sum(_lengths(case)), case['batch'], case['heads'], case['depth']
    seen = 0.9 * rows * (B - 1 if B > 1 else 1) / B if case['mask'] else rows
    return {'bytes': 2.0 * es * seen * case['kv_heads'] * D + 8.0 * B * H * D + 4.0 * rows / case['page'] + (4.0 * rows if case['mask'] else 0.0),
            'flops': 4.0 * seen * H * D}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    page = case['page']
    if case['op'] == 'plan':
        return None
    if case['op'] == 'write':
        live = s['slots'] >= 0
        slot, Hk, D = s['slots'][live].long(), case['kv_heads'], case['depth']
        out = {}
        for name in ('k', 'v'):
            flat = s[name + '_cache'].double().transpose(1, 2).reshape(-1, Hk, D)
            flat[slot] = s[name].double()[live].reshape(-1, Hk, D)
            out[name + '_cache'] = flat.view(-1, page, Hk, D).transpose(1, 2).contiguous()
        return out
    B, H, Hk, D = case['batch'], case['heads'], case['kv_heads'], case['depth']
    out = torch.zeros(B, Hk, H // Hk, D, dtype=torch.float64, device=DEV)
    table, lengths = s['table'].cpu(), s['lengths'].tolist()
    for b in range(B):
        n = lengths[b]
        ids = table[b, :(n + page - 1) // page].long().to(DEV)
        keep = torch.ones(n, dtype=torch.bool, device=DEV) if s['mask'] is None else s['mask'][b, :n] == 0
        if not bool(keep.any()):
            continue
        for h in range(Hk):
            k = s['k_cache'][ids, h].reshape(-1, D)[:n][keep].double()
            v = s['v_cache'][ids, h].reshape(-1, D)[:n][keep].double()
            q = s['q'][b].view(Hk, H // Hk, D)[h].double()
            out[b, h] = torch.softmax(q @ k.T / D ** 0.5, -1) @ v
    return out.view(B, H * D)

"""Paged decoding without a GPU: what the entry points refuse (the C ABI with pointers that are never followed, the Python layer with
CPU tensors), the layout of the argument blocks, and models of the kernels' index arithmetic with bad pages, slots and lengths."""
import ctypes
import os
import subprocess
import warnings

import pytest
import torch

import estts
from estts import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x1000
BLOCKS = {'estts_page_plan_args': _lib.PagePlanArgs, 'estts_page_write_args': _lib.PageWriteArgs,
          'estts_paged_attention_args': _lib.PagedAttentionArgs}


@pytest.mark.parametrize('cname', sorted(BLOCKS))
def test_field_offsets_match_header_layout(tmp_path, cname):
    cls = BLOCKS[cname]
    names = [n for n, _ in cls._fields_]
    src = tmp_path / 'offsets.c'
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "estts.h"\nint main(void) {\n' +
                   ''.join(f'  printf("{n} %zu\\n", offsetof({cname}, {n}));\n' for n in names) +
                   f'  printf("sizeof %zu\\n", sizeof({cname}));\n  return 0;\n}}\n')
    exe = tmp_path / 'offsets'
    subprocess.run(['gcc', '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(exe)], check=True)
    at = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.strip().splitlines())
    assert ctypes.sizeof(cls) == int(at['sizeof'])
    for n in names:
        assert getattr(cls, n).offset == int(at[n]), n


# ---------------------------------------------------------------------------------------------------------------- C ABI refusals
def plan_block(**kw):
    f = dict(lengths=FAKE, n_new=FAKE, block_table=FAKE, ld_table=8, free_pages=FAKE, n_free=FAKE, slots=FAKE, positions=FAKE, lengths_out=FAKE,
             n_free_out=FAKE, refused=FAKE, B=4, P=8, n_pages=32, page=16, T=4, R=1)
    f.update(kw)
    return _lib.PagePlanArgs(**f)


def write_block(**kw):
    f = dict(k=FAKE, ldk=256, v=FAKE, ldv=256, k_cache=FAKE, v_cache=FAKE, s_page=4096, s_head=1024, s_row=64, slots=FAKE, T=4, heads=4, depth=64,
             page=16, n_pages=32, type=0)
    f.update(kw)
    return _lib.PageWriteArgs(**f)


def attention_block(**kw):
    f = dict(q=FAKE, ldq=256, k_cache=FAKE, v_cache=FAKE, s_page=4096, s_head=1024, s_row=64, block_table=FAKE, ld_table=8, lengths=FAKE, ctx=FAKE,
             ldo=256, scale=0.125, B=4, H=4, kv_heads=4, depth=64, page=16, n_pages=32, P=8, max_len=128, type=0)
    f.update(kw)
    return _lib.PagedAttentionArgs(**f)


@pytest.mark.parametrize('bad,word', [(dict(lengths=None), 'null'), (dict(free_pages=None), 'null'), (dict(B=0), 'shape'), (dict(T=0), 'shape'),
                                      (dict(ld_table=7), 'shape'), (dict(R=2), 'padded'), (dict(T=5000, R=0), 'scratch'),
                                      (dict(T=5000, R=0, ws=FAKE, ws_bytes=79), 'scratch'), (dict(B=5000, T=5000), 'scratch'), (dict(page=8), 'multiple of 16'), (dict(page=0), 'multiple of 16'),
                                      (dict(page=24), 'multiple of 16'), (dict(n_pages=1 << 27), '2^31'), (dict(P=1 << 27, ld_table=1 << 27), '2^31')])
def test_page_plan_refuses(bad, word):
    lib = _lib.load()
    assert lib.estts_page_plan(plan_block(**bad), None) != 0
    assert word in lib.estts_last_error().decode(), lib.estts_last_error()


@pytest.mark.parametrize('bad,word', [(dict(k=None), 'null'), (dict(slots=None), 'null'), (dict(T=0), 'shape'), (dict(depth=60), 'depth'),
                                      (dict(depth=4096), 'depth'), (dict(page=20), 'multiple of 16'), (dict(type=3), 'type'), (dict(ldk=128), 'rows'),
                                      (dict(ldv=258), 'rows'), (dict(k=FAKE + 4), 'rows'), (dict(k_cache=FAKE + 8), '16 bytes'),
                                      (dict(s_head=1022), '16 bytes'), (dict(type=1, s_page=4100), '16 bytes'), (dict(s_row=32), '16 bytes'),
                                      (dict(n_pages=1 << 27), '2^31')])
def test_page_write_refuses(bad, word):
    lib = _lib.load()
    assert lib.estts_page_write(write_block(**bad), None) != 0
    assert word in lib.estts_last_error().decode(), lib.estts_last_error()


@pytest.mark.parametrize('bad,word', [(dict(q=None), 'null'), (dict(lengths=None), 'null'), (dict(B=0), 'shape'), (dict(B=65536), 'shape'),
                                      (dict(H=6), 'shape'), (dict(depth=48), 'depth'), (dict(depth=256), 'depth'), (dict(page=12), 'multiple of 16'),
                                      (dict(type=-1), 'type'), (dict(ldq=192), 'query rows'), (dict(ldo=255), 'query rows'),
                                      (dict(q=FAKE + 8), 'query rows'), (dict(s_row=66), '16 bytes'), (dict(k_cache=FAKE + 2), '16 bytes'),
                                      (dict(max_len=-1), 'max_len'), (dict(s_row=1 << 25), '2^28'), (dict(n_pages=1 << 27), '2^31')])
def test_paged_attention_refuses(bad, word):
    lib = _lib.load()
    assert lib.estts_paged_attention(attention_block(**bad), None) != 0
    assert word in lib.estts_last_error().decode(), lib.estts_last_error()


def test_null_blocks_are_refused():
    lib = _lib.load()
    for name in ('estts_page_plan', 'estts_page_write', 'estts_paged_attention'):
        assert getattr(lib, name)(None, None) != 0 and b'null args' in lib.estts_last_error()


# ------------------------------------------------------------------------------------------------------------- Python refusals
def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def plan_call(**kw):
    f = dict(lengths=i32(4), new=i32(4), block_table=i32(4, 8), free_pages=i32(32), n_free=i32(1), page=16, slots=i32(4, 1))
    f.update(kw)
    return ops.page_plan(**f)


@pytest.mark.parametrize('bad,error', [(dict(), 'is on cpu'), (dict(new=i32(3)), 'new'), (dict(new=torch.zeros(4)), 'int32'), (dict(block_table=i32(3, 8)), 'block_table'),
                                       (dict(block_table=i32(8, 4).t()), 'block_table'), (dict(block_table=i32(4, 8).long()), 'int32'), (dict(slots=i32(3, 1)), 'slots'),
                                       (dict(slots=i32(2, 2, 1)), 'slots'), (dict(slots=i32(4, 2)[:, :1]), 'slots'), (dict(positions=i32(4)), 'positions'),
                                       (dict(lengths_out=i32(5)), 'lengths_out'), (dict(n_free=i32(2)), 'n_free'), (dict(refused=i32(4)), 'refused')])
def test_page_plan_checks_its_arguments(bad, error):
    with pytest.raises((ValueError, TypeError), match=error):
        plan_call(**bad)


def caches(**kw):
    return torch.zeros(32, 4, 16, 64, **kw), torch.zeros(32, 4, 16, 64, **kw)


@pytest.mark.parametrize('bad,error', [(dict(), 'is on cpu'), (dict(k=torch.zeros(4, 128)), 'k must be'), (dict(v=torch.zeros(5, 256)), 'v must be'),
                                       (dict(k=torch.zeros(256, 4).t()), 'k must be'), (dict(k=torch.zeros(4, 256).bfloat16()), 'float32'), (dict(slots=torch.zeros(4)), 'int32'),
                                       (dict(k_cache=torch.zeros(32, 4, 16, 64).double(), v_cache=torch.zeros(32, 4, 16, 64).double()), 'float16'),
                                       (dict(k_cache=torch.zeros(32, 4, 16, 64).half()), 'same strides'), (dict(k_cache=torch.zeros(32, 16, 4, 64).transpose(1, 2)), 'same strides'),
                                       (dict(k_cache=torch.zeros(1, 4, 16, 64).expand(32, 4, 16, 64), v_cache=torch.zeros(1, 4, 16, 64).expand(32, 4, 16, 64)), 'broadcast'),
                                       (dict(k_cache=torch.zeros(32, 4, 64, 16).transpose(2, 3), v_cache=torch.zeros(32, 4, 64, 16).transpose(2, 3)), 'contiguous')])
def test_page_write_checks_its_arguments(bad, error):
    k_cache, v_cache = caches()
    f = dict(k=torch.zeros(4, 256), v=torch.zeros(4, 256), k_cache=k_cache, v_cache=v_cache, slots=i32(4))
    f.update(bad)
    with pytest.raises((ValueError, TypeError), match=error):
        ops.page_write(**f)


@pytest.mark.parametrize('bad,error', [(dict(), 'is on cpu'), (dict(q=torch.zeros(4, 255)), 'q must be'), (dict(ctx=torch.zeros(3, 256)), 'ctx must be'),
                                       (dict(q=torch.zeros(4, 256).half()), 'float32'), (dict(heads=6), 'do not divide'), (dict(heads=0), 'do not divide'),
                                       (dict(lengths=i32(4).long()), 'int32'), (dict(block_table=i32(5, 8)), 'block_table'), (dict(max_len=0), 'max_len'),
                                       (dict(key_mask=torch.zeros(4, 127)), 'key_mask'), (dict(key_mask=torch.zeros(4, 128, dtype=torch.bool)), 'key_mask'),
                                       (dict(key_mask=torch.zeros(3, 128)), 'key_mask')])
def test_paged_attention_checks_its_arguments(bad, error):
    k_cache, v_cache = caches()
    f = dict(q=torch.zeros(4, 256), k_cache=k_cache, v_cache=v_cache, block_table=i32(4, 8), lengths=i32(4), ctx=torch.zeros(4, 256), heads=4)
    f.update(bad)
    with pytest.raises((ValueError, TypeError), match=error):
        ops.paged_attention(**f)


def test_caches_without_heads_or_rows_are_refused():
    for shape, error in (((32, 0, 16, 64), 'do not divide'), ((32, 4, 0, 64), 'max_len')):
        with pytest.raises(ValueError, match=error):
            ops.paged_attention(torch.zeros(4, 256), torch.zeros(shape), torch.zeros(shape), i32(4, 8), i32(4), torch.zeros(4, 256), 4)


def test_pages_must_be_a_multiple_of_sixteen_rows():
    lib = _lib.load()
    for page in (1, 8, 15, 17, 40):
        assert lib.estts_page_plan(plan_block(page=page), None) != 0 and b'multiple of 16' in lib.estts_last_error()


# ------------------------------------------------------------------------------------------- models of the kernels' index arithmetic
# The formulas restate csrc/paged.hip; a kernel change that moves an index has to move it here too.
def divide(x, d, bits):
    """Divisor: x / d for x below 2^bits, a product of 32-bit numbers and a shift."""
    s = (d - 1).bit_length()
    m = -(-(1 << (bits + s)) // d)
    assert 0 < m < 2 ** 32 and bits + s < 64 and x < 2 ** bits
    return x * m >> (bits + s)


def pages(x, page):
    """PageSize: x / page for x below 2^32."""
    return divide(x >> 4, page // 16, 28)


@pytest.mark.parametrize('bits', [28, 30])
def test_divisions_are_exact(bits):
    g = torch.Generator().manual_seed(bits)
    ds = list(range(1, 70)) + [100, 127, 128, 129, 255, 256, 257, 1000, 4095, 4096, 65535, 2 ** 20 - 1, 2 ** 20 + 1, 2 ** 26, 2 ** bits - 1]
    ds += torch.randint(1, 2 ** 24, (50,), generator=g).tolist()
    for d in ds:
        top = 2 ** bits - 1
        xs = [0, 1, d - 1, d, d + 1, top, top - 1, top // d * d, max(top // d * d - 1, 0)] + torch.randint(0, 2 ** bits, (50,), generator=g).tolist()
        xs += [k * d + e for k in (2, 3, top // d // 2) for e in (-1, 0, 1)]
        for x in xs:
            if 0 <= x <= top:
                assert divide(x, d, bits) == x // d, (x, d)
    for page in (16, 32, 48, 64, 112, 1600, 2 ** 30):
        for x in (0, 1, page - 1, page, page + 1, 2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 5 * page - 1, 5 * page):
            if x < 2 ** 32:
                assert pages(x, page) == x // page


def request_rows(length, P, page, max_len):
    return min(max(length, 0), P * page, max_len)


def parts_of(lengths, target, unit):
    """PagedPart: for every part the segments (request, first unit, units, units of the request, place or None) it works through, and
    where the join finds each request (first part, number of parts)."""
    units = [max(-(-n // unit), 1) for n in lengths]
    total = sum(units)
    n_parts = min(target, total)
    share = divide(total, target, 30) if total >= target else 1
    extra = total - share * n_parts
    part_of = lambda x: int(((x + 1.0) * n_parts - 1.0) / total)
    line, parts, items = 0, [], {}
    starts = []
    for n in units:
        starts.append(line)
        line += n
    for k in range(n_parts):
        lo = k * share + divide(k * extra, target, 30)
        hi = lo + share + divide((k + 1) * extra, target, 30) - divide(k * extra, target, 30)
        assert (lo, hi) == (k * total // n_parts, (k + 1) * total // n_parts)
        b = max(i for i, s in enumerate(starts) if s <= lo)
        off, left, at, segments = lo - starts[b], hi - lo, lo, []
        while left > 0:
            take = min(units[b] - off, left)
            whole = take == units[b]
            segments.append((b, off, take, units[b], None if whole else 2 * k + (off == 0)))
            if off == 0:
                items[b] = (k, 1 if whole else part_of(at + units[b] - 1) - k + 1)
            left, at, off, b = left - take, at + take, 0, b + 1
        parts.append(segments)
    return parts, items


@pytest.mark.parametrize('lengths', [[0], [1], [131071], [5000, 0, 0, 1, 300, 128, 129], [100] * 300, [0] * 7, [3000] + [1] * 700 + [2500], list(range(0, 4000, 37))])
@pytest.mark.parametrize('target', [1, 2, 32, 64, 256])
@pytest.mark.parametrize('unit', [64, 128])
def test_parts_cover_every_row_once_and_the_join_finds_them(lengths, target, unit):
    parts, items = parts_of(lengths, target, unit)
    seen, places = {}, {}
    for k, segments in enumerate(parts):
        assert segments
        for b, off, take, n, place in segments:
            for u in range(off, off + take):
                assert (b, u) not in seen
                seen[b, u] = k
            if place is not None:
                assert 0 <= place < 2 * target and place not in places          # (two places a part, each used once)
                places[place] = b
    for b, rows in enumerate(lengths):
        n = max(-(-rows // unit), 1)
        assert all((b, u) in seen for u in range(n)) and (b, n) not in seen
        first, count = items[b]
        assert (first, count) == (seen[b, 0], seen[b, n - 1] - seen[b, 0] + 1)
        if count > 1:                               # what paged_join_kernel reads
            read = [2 * first + 1] + [2 * (first + s) for s in range(1, count)]
            assert [places[x] for x in read] == [b] * count
    # equal parts: no two differ by more than a unit
    sizes = [sum(t for _, _, t, _, _ in s) for s in parts]
    assert max(sizes) - min(sizes) <= 1


@pytest.mark.parametrize('halves,waves', [(1, 4), (2, 4), (1, 8), (2, 8)])
@pytest.mark.parametrize('page', [16, 48, 64])
@pytest.mark.parametrize('P,max_len,begin,end', [(1, 16, 0, 1), (3, 40, 0, 40), (70, 1000, 0, 1000), (70, 1111, 512, 1111), (700, 9000, 4096, 9000)])
def test_page_walk_stays_inside_table_and_pages(halves, waves, page, P, max_len, begin, end):
    """Every table entry that PageWalk reads lies in the request's row of the table, every half of a tile in one page, and the lanes hold
    the half that locate() asks for."""
    max_len = min(max_len, P * page)
    end = min(end, max_len)
    tile, per_block = 16 * halves, 64 // halves
    n_tiles = max(-(-(end - begin) // tile), 0)
    half_row = lambda block, lane, wave: begin + ((block * per_block + lane // halves) * waves + wave) * tile + 16 * (lane % halves)
    for wave in range(waves):
        mine = (n_tiles - wave + waves - 1) // waves if n_tiles > wave else 0
        for block in range(max(mine - 1, 0) // per_block + 3):
            for lane in (0, 1, 2, 31, 62, 63):
                assert 0 <= min(half_row(block, lane, wave), max_len - 1) // page < P
        for it in range(mine):
            for s in range(halves):
                lane = (it % per_block) * halves + s
                r = half_row(it // per_block, lane, wave)
                assert r == begin + (it * waves + wave) * tile + 16 * s
                assert r % page + 15 < page or r % page + 16 == page           # (sixteen rows of one page)


@pytest.mark.parametrize('entry', [-2 ** 31, -1, 7, 8, 2 ** 31 - 1])
def test_pages_and_slots_that_do_not_exist_reach_no_memory(entry):
    """place() and page_write_kernel: an id or slot outside the cache is never turned into an address."""
    n_pages, page = 7, 16
    there = 0 <= entry < n_pages
    assert not there                                                            # (place: offset -1, locate: row 0 of page 0, rows left out)
    for slot in (entry, entry & 0xFFFFFFFF):
        assert (slot & 0xFFFFFFFF) >= n_pages * page or 0 <= slot < n_pages * page
    assert ((-1) & 0xFFFFFFFF) >= n_pages * page


@pytest.mark.parametrize('depth,esize', [(32, 2), (64, 2), (128, 2), (32, 4), (64, 4), (128, 4)])
def test_lane_loads_cover_each_row_once(depth, esize):
    """feature_of and the byte offsets of the loads: the 16 lanes of a row read every byte of it once, and element e of lane r is feature
    feature_of(r, e); of K, lane (i, g) of load x reads bytes 16 g + 64 x .. + 15."""
    nv = depth // 16
    run = nv if nv * esize < 16 else 16 // esize
    feature = lambda r, e: (e // run) * (16 * run) + r * run + e % run
    assert sorted(feature(r, e) for r in range(16) for e in range(nv)) == list(range(depth))
    for r in range(16):
        for e in range(nv):
            load = e // run
            assert feature(r, e) * esize == r * run * esize + 256 * load + (e % run) * esize
    k_bytes = sorted(b for g in range(4) for x in range(depth * esize // 64) for b in range(16 * g + 64 * x, 16 * g + 64 * x + 16))
    assert k_bytes == list(range(depth * esize))
    # buffer range of a half: the last byte read is the last of its sixteenth row
    row_bytes = depth * esize + 32
    half_bytes = 15 * row_bytes + depth * esize
    last_v = 4 * 3 * row_bytes + 15 * run * esize + 256 * ((nv - 1) // run) + 3 * row_bytes + run * esize
    last_k = 15 * row_bytes + 16 * 3 + 64 * (depth * esize // 64 - 1) + 16
    assert last_v == last_k == half_bytes


@pytest.mark.parametrize('B,heads,kv_heads,depth,max_len,type,cut', [
    (1, 4, 4, 64, 1024, 0, False), (1, 4, 4, 64, 1025, 0, True), (1, 4, 4, 128, 512, 0, False), (1, 4, 4, 128, 513, 0, True), (8, 4, 4, 128, 600, 0, True),
    (9, 4, 4, 128, 600, 0, False), (1, 12, 4, 128, 256, 0, False), (1, 12, 4, 128, 257, 0, True), (1, 32, 8, 128, 513, 1, True), (8, 32, 8, 128, 513, 2, True),
    (9, 32, 8, 128, 513, 1, False), (1, 8, 8, 128, 1000, 1, False), (1, 64, 1, 64, 1000, 2, False), (32, 8, 8, 64, 2048, 0, False), (32, 8, 8, 64, 2049, 0, True),
    (31, 8, 8, 64, 2048, 0, True), (128, 8, 8, 64, 2048, 0, True), (1, 600, 600, 32, 5000, 1, True)])
def test_which_calls_are_cut(B, heads, kv_heads, depth, max_len, type, cut):
    lib = _lib.load()
    nbytes = lib.estts_paged_attention_ws_bytes(B, heads, kv_heads, depth, max_len, type)
    parts = max(1, 256 // (kv_heads * -(-heads // kv_heads // 16)))
    assert nbytes == (2 * parts * heads * (depth + 2) * 4 + 8 * B if cut else 0)


# ---------------------------------------------------------------------------------- where the kernels' addresses lie, bad ids among them
def half_at(entry, r, page, n_pages, max_len, s_page, s_row):
    """PageWalk: the byte (here: element) offset of the sixteen rows from r on in a page named `entry`, through place()'s two 32-bit halves and
    locate(); (offset, whether they count)."""
    there = entry >= 0 and entry < n_pages and r < max_len
    x = entry * s_page + (r - r // page * page) * s_row if there else -1
    lo, hi = x & 0xFFFFFFFF, (x >> 32) & 0xFFFFFFFF
    hi -= (hi & 0x80000000) << 1
    return ((hi & 0xFFFFFFFF) << 32 | lo, True) if hi >= 0 else (0, False)


def slot_at(slot, h, page, n_pages, s_page, s_head, s_row):
    """page_write_kernel: the element a row's head goes to, or None."""
    slot &= 0xFFFFFFFF
    return None if slot >= n_pages * page else slot // page * s_page + h * s_head + slot % page * s_row


STRIDES = {'head': lambda Hk, page, D: (Hk * page * D, page * D, D), 'token': lambda Hk, page, D: (page * Hk * D, D, Hk * D),
           'gaps': lambda Hk, page, D: ((Hk + 1) * (page + 3) * (D + 16), (page + 3) * (D + 16), D + 16)}


@pytest.mark.parametrize('order', sorted(STRIDES))
@pytest.mark.parametrize('n_pages,page,Hk,D', [(1, 16, 1, 32), (7, 16, 3, 64), (7, 48, 2, 128), (131113, 64, 4, 128)])
def test_addresses_lie_in_the_cache_or_are_not_taken(n_pages, page, Hk, D, order):
    """Every id and slot, those at and past the ends of the cache among them: what the attention loads is sixteen rows that the cache has
    (row 0 of page 0 in the place of rows that do not count), what the write stores is a row that it has; valid ones are all taken."""
    s_page, s_head, s_row = STRIDES[order](Hk, page, D)
    end = (n_pages - 1) * s_page + (Hk - 1) * s_head + (page - 1) * s_row + D           # one past the last element
    heads = (0, Hk - 1)
    max_len = 5 * page - 7
    for entry in (-2 ** 31, -n_pages, -1, 0, 1, n_pages // 2, n_pages - 1, n_pages, n_pages + 1, 2 ** 31 - 1):
        for r in list(range(0, 5 * page, 16)) + [5 * page, 1 << 30]:
            at, counts = half_at(entry, r, page, n_pages, max_len, s_page, s_row)
            assert counts == (0 <= entry < n_pages and r < max_len)
            assert at == (entry * s_page + r % page * s_row if counts else 0)
            for h in heads:
                assert 0 <= at + h * s_head and at + h * s_head + 15 * s_row + D <= end
    total = n_pages * page
    for slot in (-2 ** 31, -total, -page, -1, 0, 1, page - 1, page, total // 2, total - page, total - 1, total, total + 1, 2 ** 31 - 1):
        for h in heads:
            at = slot_at(slot, h, page, n_pages, s_page, s_head, s_row)
            assert (at is not None) == (0 <= slot < total)
            assert at is None or (0 <= at and at + D <= end and at == slot // page * s_page + h * s_head + slot % page * s_row)


# -------------------------------------------------------------------------------------------------------------- the C++ module
def test_the_cpp_module_is_built_for_this_torch():
    assert _lib.load_host() and _lib.load_host().built_for == (torch.__version__, _lib.ABI_VERSION)


@pytest.mark.parametrize('why', ['missing', 'not a module', 'another torch', 'another ABI', 'an older build'])
def test_without_a_usable_cpp_module_calls_take_the_python_path(monkeypatch, tmp_path, why):
    """Said once, not raised: the kernels are all there without it."""
    real = _lib.load_host()
    monkeypatch.setattr(_lib, '_host', None)
    if why in ('missing', 'not a module'):
        monkeypatch.setattr(_lib, '_PKG', str(tmp_path))
        if why == 'not a module':
            (tmp_path / '_hostops.so').write_bytes(b'no library')
    elif why == 'an older build':
        monkeypatch.delattr(real, 'built_for')
        monkeypatch.setattr('importlib.util.module_from_spec', lambda spec: real)
        monkeypatch.setattr('importlib.machinery.ExtensionFileLoader.exec_module', lambda self, mod: None)
    else:
        monkeypatch.setattr(*((torch, '__version__', '1.0') if why == 'another torch' else (_lib, 'ABI_VERSION', 0)))
    with pytest.warns(RuntimeWarning, match='from Python'):
        assert ops._issue() is None
    with warnings.catch_warnings():
        warnings.simplefilter('error')
        assert ops._issue() is None and _lib._host is False
        with pytest.raises((ValueError, TypeError)):                # (the Python path, and its checks)
            ops.paged_attention(*[torch.zeros(1)] * 6, 1)


# ------------------------------------------------------------------------------------------------- sizes that do not fit 32 bits
def meta(*shape, dtype=torch.int32):
    return torch.empty(*shape, dtype=dtype, device='meta')


@pytest.mark.parametrize('name,call', [
    ('rows', lambda: ops.page_plan(meta(3), meta(3), meta(3, 8), meta(32), meta(1), 16, meta(2 ** 32 + 5))),
    ('pages', lambda: ops.page_plan(meta(3), meta(3), meta(3, 8), meta(2 ** 32 + 5), meta(1), 16, meta(4))),
    ('requests', lambda: ops.page_plan(meta(2 ** 32 + 3), meta(2 ** 32 + 3), meta(2 ** 32 + 3, 8), meta(32), meta(1), 16, meta(4))),
    ('pages_of_a_request', lambda: ops.page_plan(meta(3), meta(3), meta(3, 2 ** 32 + 8), meta(32), meta(1), 16, meta(4))),
    ('page', lambda: ops.page_plan(meta(3), meta(3), meta(3, 8), meta(32), meta(1), 2 ** 32 + 16, meta(4))),
    ('rows', lambda: ops.page_write(*[meta(2 ** 32 + 5, 64, dtype=torch.float32)] * 2, *[meta(4, 2, 16, 32, dtype=torch.float32)] * 2, meta(2 ** 32 + 5))),
    ('pages', lambda: ops.page_write(*[meta(5, 64, dtype=torch.float32)] * 2, *[meta(2 ** 32 + 4, 2, 16, 32, dtype=torch.float32)] * 2, meta(5))),
    ('requests', lambda: ops.paged_attention(meta(2 ** 32 + 1, 64, dtype=torch.float32), *[meta(4, 2, 16, 32, dtype=torch.float32)] * 2, meta(2 ** 32 + 1, 8),
                                             meta(2 ** 32 + 1), meta(2 ** 32 + 1, 64, dtype=torch.float32), 2, max_len=64)),
    ('pages_of_a_request', lambda: ops.paged_attention(meta(1, 64, dtype=torch.float32), *[meta(4, 2, 16, 32, dtype=torch.float32)] * 2, meta(1, 2 ** 32 + 1),
                                                       meta(1), meta(1, 64, dtype=torch.float32), 2, max_len=64))])
def test_sizes_past_32_bits_are_refused(name, call):
    """As int32 fields of the argument block 2**32 + 5 rows would be five: the plan of the others would stay as it was."""
    with pytest.raises(ValueError, match=rf': {name} must stay below 2\*\*31'):
        call()

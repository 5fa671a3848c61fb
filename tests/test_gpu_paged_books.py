"""GPU: block tables, slot maps and the writing of new tokens, against Python's own books."""
import pytest
import torch

from aotriton_b200 import paged

pytestmark = pytest.mark.gpu


def books(table, lengths, new, free, page, total, taken=0):
    """What block_tables gives, one token after another."""
    table = [list(r) for r in table]
    slots, ends = [], [0]
    for z, (n, m) in enumerate(zip(lengths, new)):
        n, m = max(n, 0), max(m, 0)
        for p in range(n, n + m):
            i = p // page
            if i >= len(table[z]):
                slots.append(-1)
                continue
            if p % page == 0:
                table[z][i] = free[taken] if taken < len(free) else -1
                taken += 1
            slots.append(-1 if table[z][i] < 0 else table[z][i] * page + p % page)
        ends.append(ends[-1] + m)
    return table, (slots + [-1] * (total - len(slots)))[:total], ends, [max(n, 0) + max(m, 0) for n, m in zip(lengths, new)], taken


def run(lengths, new, page, width, free, extra=0, taken=None, seed=0):
    b = len(lengths)
    g = torch.Generator().manual_seed(seed)
    table = torch.randint(0, 1000, (b, width), generator=g)
    for z, n in enumerate(lengths):
        table[z, -(-max(n, 0) // page):] = -5
    total = sum(max(m, 0) for m in new) + extra
    dev = torch.full((b, width + 3), 77, dtype=torch.int32, device="cuda")
    rows = dev[:, :width]
    rows.copy_(table)
    cursor = None if taken is None else torch.tensor([taken], dtype=torch.int32, device="cuda")
    args = (rows, *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, new, free)), page, total)
    r = paged.block_tables(*args, taken=cursor)
    want = books(table.tolist(), lengths, new, free, page, total, taken or 0)
    for _ in range(2):      # (again on the same arguments: the same)
        assert rows.tolist() == want[0] and (dev[:, width:] == 77).all()
        assert r.slots.tolist() == want[1] and r.cu_seqlens.tolist() == want[2] and r.lengths.tolist() == want[3] and r.taken.tolist() == [want[4]]
        r = paged.block_tables(*args, taken=cursor)


@pytest.mark.parametrize("page", [1, 3, 16, 64])
def test_small_batches(page):
    run([0, 1, page - 1, page, page + 1, 100], [1] * 6, page, 120, list(range(2000, 2100)))
    run([0, 5, 0, 70], [0, 33, 200, 1], page, 250, list(range(2400, 2000, -1)), extra=10)
    run([7], [0], page, 10, [], extra=3)
    run([0], [1], page, 1, [9])


def test_many_sequences_and_long_prompts():
    lengths = [(i * 7919) % 300 for i in range(1000)]
    new = [(i * 104729) % 5 if i % 50 else 3000 for i in range(1000)]
    run(lengths, new, 16, 250, list(range(10000, 16000)))
    run([0, 3], [9000, 8000], 64, 200, list(range(500)), extra=5000)
    run([0] * 700, [0] * 699 + [1], 16, 2, [3])
    run([0] * 700, [0] * 700, 16, 2, [3], extra=1)


def test_too_little_room():
    run([0, 30, 5], [100, 100, 100], 16, 5, list(range(50)))      # rows too short
    run([0, 30, 5], [40, 40, 40], 16, 12, [8, 9, 10])             # free list used up
    run([0, 30, 5], [40, 40, 40], 16, 12, [], extra=1)
    run([0, 4], [20, 20], 16, 4, list(range(10)), taken=3)
    run([0, 4], [20, 20], 16, 4, list(range(10)), taken=9)
    run([-3, 4], [20, -2], 16, 4, list(range(10)))
    run([5, 5], [3, 3], 16, 0, [1])


def test_no_sequences_and_no_room_for_tokens():
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    r = paged.block_tables(torch.empty(0, 4, dtype=torch.int32, device="cuda"), empty, empty, empty, 16, 5)
    assert r.slots.tolist() == [-1] * 5 and r.cu_seqlens.tolist() == [0] and r.taken.tolist() == [0] and r.lengths.numel() == 0
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    n, m = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 0], [40, 5]))
    r = paged.block_tables(table, n, m, torch.arange(9, dtype=torch.int32, device="cuda"), 16, 20)      # less than 45
    assert r.slots.tolist() == list(range(20)) and r.cu_seqlens.tolist() == [0, 40, 45] and table.tolist() == [[0, 1, -1, -1], [-1] * 4]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,dv", [(128, 128), (64, 72), (5, 3), (6, 2), (512, 64)])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_writing(dtype, d, dv, layout):
    g = torch.Generator(device="cuda").manual_seed(1)
    for tokens, hk, page, offset in ((1, 1, 16, 0), (37, 3, 5, 0), (500, 2, 16, 0), (40, 2, 16, 1)):
        pages = tokens // page + 2

        def cache(w):
            c = torch.randn(pages, hk, page, w + offset, generator=g, device="cuda").to(dtype)
            return (c.transpose(1, 2) if layout == "hnd" else c.transpose(1, 2).contiguous())[..., offset:]

        kc, vc = cache(d), cache(dv)
        both = torch.randn(tokens, hk, d + dv + offset, generator=g, device="cuda").to(dtype)
        k, v = both[..., offset:offset + d], both[..., offset + d:]
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
        slots[::4] = -1
        if tokens > 2:
            slots[1] = pages * page      # behind the cache
        want = [c.clone() for c in (kc, vc)]
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                want[0][s // page, s % page], want[1][s // page, s % page] = k[t], v[t]
        paged.paged_write(k, v, kc, vc, slots)
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
        kc2 = torch.zeros_like(kc)
        paged.paged_write(k, None, kc2, None, slots)
        paged.paged_write(k.transpose(1, 2).contiguous().transpose(1, 2), None, kc, None, slots)
        assert torch.equal(kc, want[0])


def test_latent_rows_and_versions():
    cache = torch.zeros(4, 16, 576, device="cuda", dtype=torch.bfloat16)
    latent, rope = torch.randn(3, 512, device="cuda").bfloat16(), torch.randn(3, 64, device="cuda").bfloat16()
    was = cache._version
    paged.paged_write(latent[:, None], rope[:, None], cache[:, :, None, :512], cache[:, :, None, 512:], torch.tensor([5, 63, 20], device="cuda"))
    assert torch.equal(cache.view(64, 576)[[5, 63, 20]], torch.cat([latent, rope], 1)) and cache._version > was
    assert int(cache.view(64, 576).any(1).sum()) == 3
    paged.paged_write(latent[:0, None], None, cache[:, :, None, :512], None, torch.empty(0, dtype=torch.int64, device="cuda"))


def test_a_step_of_everything_captured():
    """Books, writing and attention as one captured step, replayed: the lengths advance on the device."""
    b, hq, hk, d, page = 3, 8, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    table = torch.full((b, 8), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(b, dtype=torch.int32, device="cuda")
    taken = torch.zeros(1, dtype=torch.int32, device="cuda")
    free = torch.randperm(30, generator=g, device="cuda").int()
    new = torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda")
    kc, vc = (torch.full((30, page, hk, d), float("nan"), device="cuda", dtype=torch.float16) for _ in range(2))
    q, k, v = (torch.randn(b, n, d, generator=g, device="cuda").half() for n in (hq, hk, hk))

    def step():
        s = paged.block_tables(table, lengths, new, free, page, b, taken)
        paged.paged_write(k, v, kc, vc, s.slots)
        out = paged.paged_attention(q[:, :, None], kc, vc, table, s.lengths)
        lengths.copy_(s.lengths)
        taken.copy_(s.taken)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    lengths.zero_(), taken.zero_(), table.fill_(-1), kc.fill_(float("nan")), vc.fill_(float("nan"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    keys, values = [], []
    for i in range(40):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        keys.append(k.clone()), values.append(v.clone())
        graph.replay()
        kk, vv = torch.stack(keys, 2).double(), torch.stack(values, 2).double()
        for z in range(2):
            x = torch.einsum("hd,hnd->hn", q[z].double(), kk[z].repeat_interleave(hq // hk, 0)) * d ** -0.5
            want = torch.einsum("hn,hnd->hd", torch.softmax(x, -1), vv[z].repeat_interleave(hq // hk, 0))
            # weights and output rounded once each to 11 bits, values below 6
            assert (out[z, :, 0].double() - want).abs().max() <= 2 * 2.0 ** -11 * 6
        assert (out[2] == 0).all()
    assert lengths.tolist() == [40, 40, 0] and taken.tolist() == [6]
    assert table[:2, :3].min() >= 0 and (table[:, 3:] == -1).all() and (table[2] == -1).all()

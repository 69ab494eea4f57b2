"""A server's steps: positions turned, room made, rows added in 4 bits, attended to; sequences that fork, give drafts back, and whose pages are
moved together.  Compared with attention in 64 bits over the rows that the definitions say are there."""
import pytest
import torch

from tests.kv_plain_four import coded4, values4
from tests.test_gpu_kv_rows import i32

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


class Server:
    """One layer, and beside it every sequence's rows as lists on the CPU."""

    def __init__(self, dtype, heads, group, dim, page, pages, width, seed):
        import ferrolm_b200 as fv

        self.c = fv.KvCache(pages, heads, dim, page_size=page, dtype=dtype, kind="int4x32")
        self.pages, self.rotary = fv.KvPages(self.c), fv.Rotary(dim, part=dim // 2, layout="pairs", factor=4.0, original=64)
        self.heads, self.group, self.dim, self.dtype, self.width = heads, group, dim, dtype, width
        self.g = torch.Generator().manual_seed(seed)
        self.table, self.rows = torch.full((0, width), -1, dtype=torch.int32, device="cuda"), []

    def start(self, n):
        self.table, self.rows = torch.full((n, self.width), -1, dtype=torch.int32, device="cuda"), [([], []) for _ in range(n)]

    def lens(self):
        return i32([len(r[0]) for r in self.rows]).cuda()

    def step(self, new):
        """Adds `new` rows of random projections to the sequences and checks what they attend to."""
        H, G, D = self.heads, self.group, self.dim
        x = torch.randn((sum(new), H * (G + 2), D), generator=self.g).to(self.dtype).cuda()
        q, k, v = x.split([H * G, H, H], 1)
        before, more = self.lens(), i32(new).cuda()
        after = before + more
        cu = None if set(new) == {1} else i32([0] + torch.tensor(new).cumsum(0).tolist()).cuda()
        q, k = self.rotary.rotate(q, k, lens=after, cu=cu)
        self.pages.extend(self.table, before, more)
        assert int(self.pages.missing) == 0
        self.c.add(k, v, self.table, after, cu=cu)
        out = self.c.attend(q, self.table, after, cu=cu).cpu().double().view(-1, H, G, D)
        kk, vv, qq, r = (values4(*coded4(k.cpu().double())), values4(*coded4(v.cpu().double())), q.cpu().double().view(-1, H, G, D), 0)
        for b, n in enumerate(new):
            for _ in range(n):
                ks, vs = self.rows[b]
                ks.append(kk[r]), vs.append(vv[r])
                a, w = torch.stack(ks), torch.stack(vs)
                s = torch.einsum("hgd,nhd->hgn", qq[r], a) * D**-0.5
                want = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), w)
                # weights off by 2^-10 of themselves and by their scores' 32 bits, results by half a step: of the largest value each
                assert (out[r] - want).abs().max() <= (2.0**-10 + 2.0**-14 + torch.finfo(self.dtype).eps / 2) * w.abs().max(), (b, len(ks))
                r += 1


@pytest.mark.parametrize("dtype,heads,group,dim,page", [(BF, 2, 4, 128, 16), (FP, 1, 3, 96, 32), (BF, 2, 8, 64, 64)])
def test_sequences_that_branch_and_move(dtype, heads, group, dim, page):
    s = Server(dtype, heads, group, dim, page, 64, 12, dim)
    s.pages.refs[3:40:5] = 1  # pages of somebody else
    s.start(3)
    s.step([page + 7, 2 * page, 5])
    for turn in range(4):
        s.step([1] * len(s.rows))
        parents = torch.randint(0, len(s.rows), (3 + turn % 2,), generator=s.g).tolist()
        children = s.pages.fork(s.table, s.lens(), i32(parents).cuda())
        s.pages.free(s.table)
        s.table, s.rows = children, [(list(s.rows[b][0]), list(s.rows[b][1])) for b in parents]
        s.step([1 + (turn + b) % 6 for b in range(len(parents))])  # drafts, of which some are given back
        s.rows = [(k[: len(k) - b % 3], v[: len(v) - b % 3]) for b, (k, v) in enumerate(s.rows)]
        s.pages.free(s.table, s.lens())
        if turn % 2:
            held = int((s.pages.refs > 0).sum())
            s.pages.compact(s.table)
            assert int(s.pages.used) == held and int(s.table.max()) < held
    s.step([40] + [1] * (len(s.rows) - 1))
    s.pages.free(s.table)
    assert int(s.pages.refs.sum()) == int((s.pages.refs > 0).sum()) == 8


def test_pages_behind_4_gb():
    """A sequence on the last pages of a cache whose keys are more than 2^32 bytes: written, read back, attended to, copied."""
    import ferrolm_b200 as fv

    heads, dim, page = 8, 128, 128
    pages = (1 << 32) // (heads * page * dim // 2) + 20
    c = fv.KvCache(pages, heads, dim, page_size=page, kind="int4x32")
    low = fv.KvCache(8, heads, dim, page_size=page, kind="int4x32")
    p = fv.KvPages(c)
    p.refs[: pages - 4] = 1
    table, lens, n = torch.full((1, 4), -1, dtype=torch.int32, device="cuda"), i32([300]).cuda(), 300
    p.extend(table, i32([0]).cuda(), lens)
    assert table.tolist() == [[pages - 4, pages - 3, pages - 2, -1]]
    rows, cu = torch.randn((n, heads * 6, dim)).to(BF).cuda(), i32([0, n]).cuda()
    q, k, v = rows.split([heads * 4, heads, heads], 1)
    near = i32([[5, 0, 2, -1]]).cuda()
    c.add(k, v, table, lens, cu=cu), low.add(k, v, near, lens, cu=cu)
    for a, b in zip(c.vectors(table, lens, cu=cu, rows=n), low.vectors(near, lens, cu=cu, rows=n)):
        assert torch.equal(a, b)
    for at, start in ((slice(0, n), cu), (slice(n - 1, n), None)):
        assert torch.equal(c.attend(q[at], table, lens, cu=start), low.attend(q[at], near, lens, cu=start))
    p.refs[7] = 0
    p.compact(table)
    assert table.tolist() == [[pages - 4, pages - 3, 7, -1]]
    assert torch.equal(c.attend(q, table, lens, cu=cu), low.attend(q, near, lens, cu=cu))


def test_two_servers_on_two_streams():
    """Nothing is shared between caches, their pages and turns: the steps of two at the same time are those of each alone."""
    import ferrolm_b200 as fv

    def make():
        c = fv.KvCache(200, 2, 128, page_size=16, kind="int4x32")
        return c, fv.KvPages(c), torch.full((4, 30), -1, dtype=torch.int32, device="cuda")

    rotary, x = fv.Rotary(128), [torch.randn((20, 4, 16, 128)).to(BF).cuda() for _ in range(2)]

    def run(c, pages, table, x):
        got, lens = [], torch.zeros(4, dtype=torch.int32, device="cuda")
        for n in range(20):
            pages.extend(table, lens, torch.ones_like(lens))
            lens = lens + 1
            q, k, v = x[n].split([12, 2, 2], 1)
            q, k = rotary.rotate(q, k, lens=lens)
            c.add(k, v, table, lens)
            got.append(c.attend(q, table, lens))
            if n == 9:
                last, table = table, pages.fork(table, lens, i32([1, 1, 0, 3]).cuda())
                pages.free(last)
        return torch.stack(got), table

    alone = [run(*make(), y) for y in x]
    servers, streams = [make() for _ in x], [torch.cuda.Stream() for _ in x]
    torch.cuda.synchronize()
    together = []
    for server, y, s in zip(servers, x, streams):
        with torch.cuda.stream(s):
            together.append(run(*server, y))
    torch.cuda.synchronize()
    for a, b in zip(alone, together):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("new", [1, 24])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0**-130, 40.0])
def test_scales_of_any_sign_and_size(new, scale):
    from tests.test_gpu_kv_attend import check, queries
    from tests.test_gpu_kv_four import pair
    from tests.test_gpu_kv_rows import batch

    c, p = pair(40, 2, 96, 16, FP)
    table, lens, cu = batch(2, 18, 40, 2), [280, 41], None if new == 1 else i32([0, new, 2 * new])
    check(c, p, queries(2 * new, 2, 3, 96, FP, 3), table, lens, cu, None, scale=scale)

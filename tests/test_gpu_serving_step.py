"""A whole step of a small decoder over the paged cache, captured once: the page
tables advanced by the device, the projections, rows rotated at their positions,
keys and values written, attention, block ends.  Replayed with other row counts
each time -- prompts beside single tokens, sequences that rest, one that ends and
starts again, a step that the pool cannot hold -- and every stage of every replay
compared with its definition on the device's own inputs to it, then with the same
calls made eagerly on other tables and another cache."""
import numpy as np
import pytest

import kvad_amd as K
import test_gpu_paged as T
from test_gpu_paged_mx import MX, mx
from test_gpu_step import block_end, turned

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

H, KV, HD, N, FF, LAYERS, PAGE, SEQS, ROWS, PAGES, TABLE = 4, 2, 64, 128, 192, 2, 32, 6, 80, 10, 5
WIDTH, EPS, MAX_POS = (H + 2 * KV) * HD, 1e-6, PAGE * TABLE


def held(precision, x):
    return mx(x) if precision == MX else T.rounded(precision, x)


class Decoder:
    """Weights, tables, cache and every buffer of a step, on one context."""

    def __init__(self, ctx, precision, seed):
        rng = np.random.default_rng(seed)
        f32 = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.ctx, self.norms = ctx, [(1 + 0.2 * f32(N), 1 + 0.2 * f32(N), 1 + 0.2 * f32(N)) for _ in range(LAYERS + 1)]
        self.w = [[K.Weight.from_f32(ctx, f32(o, i) / np.float32(i ** 0.5))
                   for o, i in ((WIDTH, N), (N, H * HD), (FF, N), (FF, N), (N, FF))] for _ in range(LAYERS)]
        angle = np.arange(MAX_POS)[:, None] * 1e4 ** (-np.arange(HD // 2) / (HD // 2))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.dev = {"cos": torch.from_numpy(self.cos).cuda(), "sin": torch.from_numpy(self.sin).cuda(),
                    "norms": [[torch.from_numpy(w).cuda() for w in layer] for layer in self.norms]}
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
        buf = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
        self.t = dict(len=i32(SEQS), pages=i32(SEQS, TABLE), row_start=i32(SEQS + 1), free=i32(PAGES), n_free=i32(1), status=i32(4))
        self.table = K.PageTable(SEQS, TABLE, PAGE, PAGES, *[a.data_ptr() for a in self.t.values()])
        self.rows, self.keep, self.position = i32(SEQS), torch.full((SEQS,), -1, dtype=torch.int32, device="cuda"), i32(ROWS)
        self.slot = torch.zeros(ROWS, dtype=torch.int64, device="cuda")
        self.x0 = buf(ROWS, N)
        self.b = [dict(h=buf(ROWS, N), qkv=buf(ROWS, WIDTH), qk=buf(ROWS, (H + KV) * HD), att=buf(ROWS, H * HD), o=buf(ROWS, N),
                       x1=buf(ROWS, N), h1=buf(ROWS, N), gate=buf(ROWS, FF), up=buf(ROWS, FF), down=buf(ROWS, N), x2=buf(ROWS, N),
                       h2=buf(ROWS, N)) for _ in range(LAYERS)]
        torch.cuda.synchronize()
        self.cache = K.PagedCache(ctx, LAYERS, KV, HD, PAGES, page_size=PAGE, precision=T.PRECISIONS.get(precision, K.MXFP4))
        self.table.init_dev(ctx)
        ctx.reserve(1 << 20)  # matmuls split alike captured and not
        self.batch = self.table.batch(ROWS)
        self.ws = buf(max(self.cache.attend_ws(self.batch, H) // 4, 4))

    def step(self):
        p = lambda t: t.data_ptr()  # noqa: E731
        c, norms = self.ctx, self.dev["norms"]
        self.table.release_dev(c, p(self.keep))
        self.table.step_dev(c, p(self.rows), ROWS, p(self.position), p(self.slot))
        K.rms_norm_dev(c, p(self.x0), p(norms[0][0]), ROWS, N, EPS, p(self.b[0]["h"]))
        x = self.x0
        for l in range(LAYERS):
            b, (qkv, o, gate, up, down) = self.b[l], self.w[l]
            qkv.matmul_bt_dev(p(b["h"]), ROWS, p(b["qkv"]))
            K.rope_rows_dev(c, p(self.dev["cos"]), p(self.dev["sin"]), HD // 2, MAX_POS, p(b["qkv"]), p(self.position), ROWS, H + KV,
                            p(b["qk"]), x_stride=WIDTH)
            self.cache.push_dev(l, self.batch, p(b["qk"]) + 4 * H * HD, p(b["qkv"]) + 4 * (H + KV) * HD, k_stride=(H + KV) * HD,
                                v_stride=WIDTH)
            self.cache.attend_dev(l, self.batch, H, p(b["qk"]), p(b["att"]), q_stride=(H + KV) * HD, ws_ptr=p(self.ws),
                                  ws_bytes=4 * self.ws.numel())
            o.matmul_bt_dev(p(b["att"]), ROWS, p(b["o"]))
            K.norm_residual_dev(c, p(x), p(b["o"]), ROWS, N, EPS, p(b["x1"]), scale=0.7, pre_ptr=p(norms[l][1]), out_ptr=p(b["h1"]))
            gate.matmul_bt_dev(p(b["h1"]), ROWS, p(b["gate"]))
            up.matmul_bt_dev(p(b["h1"]), ROWS, p(b["up"]))
            K.swiglu_dev(c, p(b["gate"]), p(b["up"]), ROWS * FF)
            down.matmul_bt_dev(p(b["gate"]), ROWS, p(b["down"]))
            h2 = self.b[l + 1]["h"] if l + 1 < LAYERS else b["h2"]
            K.norm_residual_dev(c, p(b["x1"]), p(b["down"]), ROWS, N, EPS, p(b["x2"]), post_ptr=p(norms[l][2]), pre_ptr=p(norms[l + 1][0]),
                                out_ptr=p(h2))
            x = b["x2"]


@pytest.mark.parametrize("precision", [MX, "i8", "f16", "f32"])
def test_a_captured_step_of_a_decoder(precision):
    stream = torch.cuda.Stream()
    ctx, other = K.Context(0), K.Context(0)
    torch.cuda.synchronize()
    try:
        ctx.set_stream(stream.cuda_stream)
        other.set_stream(stream.cuda_stream)
        with torch.cuda.stream(stream):
            d, eager = Decoder(ctx, precision, 5), Decoder(other, precision, 5)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            d.step()
        with torch.cuda.stream(stream):
            run(g, d, eager, precision)
        del g
    finally:
        torch.cuda.synchronize()
        for c in (ctx, other):
            c.set_stream(None)
            c.close()


def run(g, d, eager, precision):
    rng = np.random.default_rng(6)
    lens, keys = [0] * SEQS, [[[np.zeros((0, KV, HD), np.float32)] * 2 for _ in range(SEQS)] for _ in range(LAYERS)]
    steps = [([40, 0, 17, 0, 1, 0], None), ([1, 33, 1, 0, 1, 0], None), ([1, 1, 0, 30, 1, 2], None), ([1, 1, 1, 1, 1, 1], None),
             ([0, 1, 60, 0, 1, 1], [0, -1, 5, -1, -1, 0]), ([70, 1, 1, 1, 1, 1], None), ([1, 1, 1, 40, 33, 0], None),  # these two need 11 and 12 pages
             ([1, 1, 1, 1, 1, 1], [-1, 2, -1, 3, -1, -1])]
    refused = 0
    for turn, (rows, keep) in enumerate(steps):
        x0 = torch.from_numpy(rng.standard_normal((ROWS, N)).astype(np.float32)).cuda()
        for e in (d, eager):
            e.rows.copy_(torch.tensor(rows))
            e.keep.copy_(torch.tensor(keep or [-1] * SEQS))
            e.x0.copy_(x0)
            for b in e.b:
                b["att"].fill_(7.0)
                b["qk"].fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        eager.step()
        torch.cuda.synchronize()
        for name in d.t:
            assert torch.equal(d.t[name], eager.t[name]), name
        for l in range(LAYERS):
            for name in d.b[l]:
                assert torch.equal(d.b[l][name], eager.b[l][name]), (turn, l, name)
        # the tables
        for s in range(SEQS):
            if keep and 0 <= keep[s] < lens[s]:
                lens[s] = keep[s]
                for l in range(LAYERS):
                    keys[l][s] = [a[:keep[s]] for a in keys[l][s]]
        pages = lambda n: -(-n // PAGE)  # noqa: E731
        free = PAGES - sum(pages(n) for n in lens)
        short = sum(pages(n + r) - pages(n) for n, r in zip(lens, rows)) > free
        refused += short
        assert d.t["status"].tolist()[:2] == [K.PageTable.SHORT if short else 0, refused]
        given = [0] * SEQS if short else rows
        lens = [n + r for n, r in zip(lens, given)]
        assert d.t["len"].tolist() == lens and d.t["row_start"].tolist() == [0] + list(np.cumsum(given))
        m = sum(given)
        pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, given)] + [np.full(ROWS - m, -1)]).astype(int)
        assert d.position.tolist() == pos.tolist()
        for l in range(LAYERS):
            b = {k: v.cpu().numpy() for k, v in d.b[l].items()}
            want = turned(b["qkv"][:m, :(H + KV) * HD].reshape(m, H + KV, HD), d.cos[pos[:m]][:, None], d.sin[pos[:m]][:, None], False)
            np.testing.assert_array_equal(b["qk"][:m], want.reshape(m, (H + KV) * HD))
            assert (b["qk"][m:] == 7).all() and (b["att"][m:] == 7).all()  # rows that no sequence has
            new_k, new_v = want[:, H:], b["qkv"][:m, (H + KV) * HD:].reshape(m, KV, HD)
            at = 0
            for s, r in enumerate(given):
                keys[l][s] = [np.concatenate([a, held(precision, n[at:at + r])]) for a, n in zip(keys[l][s], (new_k, new_v))]
                at += r
            live = [s for s in range(SEQS) if lens[s]]
            got = d.cache.read(l, K.Batch.host([lens[s] for s in live], d.t["pages"].cpu().numpy()[live], [lens[s] for s in live]))
            for i in range(2):
                np.testing.assert_array_equal(got[i], np.concatenate([keys[l][s][i] for s in live]))
            at = 0
            for s, r in enumerate(given):
                if r:
                    q = want[at:at + r, :H]
                    att, tol = T.reference(q, *keys[l][s], lens[s] - r, float(np.float32(HD ** -0.5)))
                    assert (np.abs(b["att"][at:at + r].reshape(r, H, HD) - att) <= tol).all(), (turn, l, s)
                at += r
            x = (d.x0 if l == 0 else d.b[l - 1]["x2"]).cpu().numpy()
            h2 = (d.b[l + 1]["h"] if l + 1 < LAYERS else d.b[l]["h2"]).cpu().numpy()
            for args, got_x, got_h in (((x, b["o"], None, None, 0.7, d.norms[l][1], EPS), b["x1"], b["h1"]),
                                       ((b["x1"], b["down"], d.norms[l][2], None, 1.0, d.norms[l + 1][0], EPS), b["x2"], h2)):
                want_x, tol_x, want_h, tol_h = block_end(*args)
                assert (np.abs(got_x - want_x) <= tol_x).all() and (np.abs(got_h - want_h) <= tol_h).all(), (turn, l)
    assert refused == 2

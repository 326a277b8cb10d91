"""Every address expression of the text operators' kernels (csrc/ea_mxfp4.hip, ea_gemm_mxfp4.hip, ea_attention_text.hip), evaluated on the
host over random geometries and every branch of their plans: what a lane reads or writes lies inside its tensor, workspace or LDS.  (The
256 x 256 kernel's rows: tests/test_mxfp4_rows_cpu.py.)  The expressions are written down here as they stand in the kernels; the plans
are compared with the library's own workspace sizes."""
import random

import numpy as np
import pytest

I = np.int64


def inside(what, first, size, extent):
    """[first, first + size) within [0, extent) for all of `first`."""
    first = np.asarray(first, I)
    if first.size:
        assert first.min() >= 0 and first.max() + size <= extent, (what, int(first.min()), int(first.max()) + size, extent)


def cdiv(a, b):
    return (a + b - 1) // b


# ---- storage ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", range(6))
def test_storage(seed):
    rng = random.Random(seed)
    for _ in range(40):
        per, batch = rng.randint(1, 70), rng.randint(1, 3)
        K = rng.choice([rng.randint(1, 600), 8 * rng.randint(1, 90)])
        rows, ld = per * batch, K + rng.choice([0, 0, 1, 7, 8])
        bstride = per * ld + rng.choice([0, 3, 16])
        extent = (batch - 1) * bstride + (per - 1) * ld + K                  # elements of x from its first to its last
        kt = cdiv(K, 256)
        blocks = np.arange(cdiv(rows, 32) * kt)[:, None, None]
        thread = np.arange(256)[None, :, None]
        i = np.arange(4)[None, None, :]
        tile, row = blocks % kt, blocks // kt * 32 + (thread >> 5) + 8 * i
        c = thread & 31
        k = tile * 256 + c * 8
        live = np.broadcast_to(row < rows, np.broadcast_shapes(row.shape, k.shape))
        row, k, tile, c = (np.broadcast_to(a, live.shape)[live] for a in (row, k, tile, c))
        b = row // per
        src = b * bstride + (row - b * per) * ld + k
        whole = k < K if K % 8 == 0 else k + 8 <= K
        inside("x, 8 elements", src[whole], 8, extent)
        for e in range(8):
            one = ~whole & (k + e < K) & (K % 8 != 0)
            inside("x, one element", src[one] + e, 1, extent)
        piece = tile * rows + row
        inside("codes", piece * 128 + c * 4, 4, kt * rows * 128)
        inside("scales", (piece * 8 + 2 * ((c >> 2) & 3) + (c >> 4))[(c & 3) == 0], 1, kt * rows * 8)
        written = np.unique((piece * 8 + 2 * ((c >> 2) & 3) + (c >> 4))[(c & 3) == 0])
        assert written.size == kt * rows * 8 and np.unique(piece * 128 + c * 4).size == kt * rows * 32
        # reading back: y contiguous [rows, K]
        whole = (k < K) & ((K % 8 == 0) | (k + 8 <= K))
        inside("y, 8 elements", (row * K + k)[whole], 8, rows * K)


# ---- the product -----------------------------------------------------------------------------------------------------------------------
TILES = [(256, 128, 0.75), (128, 128, 0.52), (128, 64, 0.33), (64, 64, 0.22)]
SHAPE = [(4, 2, 3, 1), (4, 2, 4, 1), (2, 2, 3, 2), (2, 2, 4, 2)]                # waves in M and N, stages, groups


def mx_plan(batch, M, N, K, from_bf16, vec):
    kt = cdiv(K, 256)
    n = dict(cfg=-1, splits=1, w4=False, code=0, scale=0, part=0)
    if from_bf16 and not (M <= 16 and vec):
        n["code"], n["scale"] = kt * batch * M * 128, cdiv(kt * batch * M * 8 + 8, 256) * 256
    if M <= 16 or (M <= 32 and N <= 8192):
        return n
    count = lambda bm, bn: cdiv(M, bm) * cdiv(N, bn) * batch
    cost = [float(cdiv(count(bm, bn), 256)) * float(np.float32(us)) for bm, bn, us in TILES]
    n["cfg"] = min(range(4), key=lambda i: (cost[i], i))
    n["w4"] = cdiv(count(256, 256), 256) * float(np.float32(1.2)) < cost[n["cfg"]]
    if n["w4"] and not from_bf16 and M % 2:
        n["scale"] = cdiv(kt * batch * M * 8 + 8, 256) * 256
    if n["w4"]:
        return n
    tiles = count(*TILES[n["cfg"]][:2])
    while n["cfg"] == 3 and tiles * n["splits"] * 2 <= 256 and kt // (n["splits"] * 2) >= 24 and n["splits"] < 16:
        n["splits"] *= 2
    if n["splits"] > 1:
        n["part"] = n["splits"] * batch * M * N * 4
    return n


def _product_sizes(rng):
    M = rng.choice([rng.randint(1, 16), rng.randint(17, 32), rng.randint(33, 300), rng.randint(300, 1500)])
    N = 8 * rng.choice([rng.randint(1, 40), rng.randint(40, 500)])
    K = rng.choice([rng.randint(1, 300), rng.randint(300, 3000), rng.randint(12000, 20000)])
    return rng.randint(1, 3), M, N, K


def test_plans_are_the_librarys(lib_built):
    from easyanimate_amd import _lib
    lib, rng = _lib.load(), random.Random(1)
    for _ in range(3000):
        batch, M, N, K = _product_sizes(rng)
        for bf16 in (0, 1):
            n = mx_plan(batch, M, N, K, bool(bf16), False)
            assert lib.ea_gemm_mxfp4_workspace_bytes(batch, M, N, K, bf16) == n["code"] + n["scale"] + n["part"], (batch, M, N, K, bf16)
        B, Hkv, group = rng.randint(1, 4), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 9, 11, 16])
        Sq, Sk, D = rng.choice([1, 2, 5, rng.randint(1, 300), rng.randint(300, 5000)]), rng.randint(1, 20000), rng.choice([64, 128])
        for docs in (0, 1):
            for causal in (False, True):         # the library asks without knowing the order: both plans have to agree
                n = attention_plan(B, Hkv * group, Hkv, Sq, Sk, D, docs, causal)
                assert lib.ea_attention_text_workspace_bytes(B, Hkv * group, Hkv, Sq, Sk, D, docs) == n["part"] + n["range"], (B, Hkv, group, Sq, Sk, D, docs, causal)


def _skinny(batch, M, N, K):
    kt = cdiv(K, 256)
    MT = 1 if M <= 16 else 2
    lane = np.arange(64)
    lr, g = lane & 15, lane >> 4
    for block in {0, cdiv(N, 16) - 1, rng_mid(cdiv(N, 16))}:
        wrow = np.minimum(block * 16 + lr, N - 1)
        for t in {0, kt - 1, kt // 2}:
            for half in (0, 64):
                inside("W codes", (t * N + wrow) * 128 + g * 16 + half, 16, kt * N * 128)
            inside("W scales", (t * N + wrow) * 8 + g * 2, 2, kt * N * 8)
            for b in range(batch):
                for i in range(MT):
                    arow = np.minimum(i * 16 + lr, M - 1)
                    piece = t * batch * M + b * M + arow
                    for half in (0, 64):
                        inside("A codes", piece * 128 + g * 16 + half, 16, kt * batch * M * 128)
                    inside("A scales", piece * 8 + g * 2, 2, kt * batch * M * 8)
                    if MT == 1 and K % 8 == 0:                               # bf16 rows, K elements apart
                        for u in range(8):
                            at = t * 256 + g * 32 + (u >> 2) * 128 + (u & 3) * 8
                            ok = at < K
                            inside("A bf16", ((b * M + arow) * K + at)[ok], 8, batch * M * K)


def rng_mid(n):
    return n // 2


def _tile(batch, M, N, K, cfg, splits):
    bm, bn, _ = TILES[cfg]
    wm, wn, ns, kg = SHAPE[cfg]
    waves, kt = wm * wn, cdiv(K, 256)
    pa, pw = bm // (8 * waves), bn // (8 * waves)
    sruns = cdiv((bm + bn) // 32, waves)
    stage = bm * 128 + bn * 128 + sruns * waves * 256
    lds = kg * ns * stage
    assert lds <= 160 * 1024 and (ns - 1) * (pa + pw + sruns) < 64
    lane = np.arange(64)
    tm_all, tn_all = cdiv(M, bm), cdiv(N, bn)
    # the block -> tile map hits every tile once
    total = tm_all * tn_all
    per = (total + 7) >> 3
    seen = set()
    for blk in range(cdiv(total, 8) * 8):
        idx = (blk & 7) * per + (blk >> 3)
        if (blk >> 3) >= per or idx >= total:
            continue
        if tm_all <= 16:
            tm, tn = idx % tm_all, idx // tm_all
        else:
            band = idx // (8 * tn_all)
            rows = min(8, tm_all - band * 8)
            local = idx - band * 8 * tn_all
            tm, tn = band * 8 + local % rows, local // rows
        seen.add((tm, tn))
    assert seen == {(a, b) for a in range(tm_all) for b in range(tn_all)}
    tiles = {(0, 0), (tm_all - 1, tn_all - 1), (0, tn_all - 1), (tm_all - 1, 0)}
    for z in range(splits):
        t0, t1 = kt * z // splits, kt * (z + 1) // splits
        assert t1 > t0
        trips = cdiv(t1 - t0, kg)
        for k in range(kg):
            own = (t1 - t0 - k + kg - 1) // kg
            assert own in (trips, trips - 1) and own >= 0
            live = [t0 + k + kg * t for t in range(own)]
            for t in {*live[:1], *live[-1:]}:
                assert t0 <= t < t1
                for tm, tn in tiles:
                    row0, col0 = tm * bm, tn * bn
                    for b in {0, batch - 1}:
                        for wave in range(waves):
                            for i in range(pa):
                                r = (wave * pa + i) * 8 + (lane >> 3)
                                ra = np.where(row0 + r < M, r, M - 1 - row0)
                                inside("A codes", (t * batch * M + b * M + row0 + ra) * 128 + (((lane & 7) ^ (r & 7)) << 4), 16, kt * batch * M * 128)
                                inside("A stage", (wave * pa + i) * 1024 + lane * 16, 16, bm * 128)
                            for i in range(pw):
                                r = (wave * pw + i) * 8 + (lane >> 3)
                                rw = np.where(col0 + r < N, r, N - 1 - col0)
                                inside("W codes", (t * N + col0 + rw) * 128 + (((lane & 7) ^ (r & 7)) << 4), 16, kt * N * 128)
                                inside("W stage", (wave * pw + i) * 1024 + lane * 16, 16, bn * 128)
                            for n in range(sruns):
                                run = wave + waves * n
                                a = run < bm // 32
                                r = (run if a else run - bm // 32) * 32 + (lane >> 1)
                                last = (M - row0 if a else N - col0) - 1
                                sv = np.minimum(r, last) * 8 + (lane & 1) * 4
                                inside("scales", sv + ((t * batch * M + b * M + row0) * 8 if a else (t * N + col0) * 8), 4,
                                       kt * (batch * M if a else N) * 8)
                                inside("scale stage", bm * 128 + bn * 128 + run * 256 + lane * 4, 4, stage)
    # fragment and scale reads of a stage, the groups' join
    lr, g = lane & 15, lane >> 4
    for wr in range(wm):
        for wc in range(wn):
            for ch in ((g ^ (lr & 7)) << 4, ((4 + g) ^ (lr & 7)) << 4):
                for f in range(bm // wm // 16):
                    inside("A fragment", (wr * (bm // wm) + lr) * 128 + f * 2048 + ch, 16, bm * 128)
                for f in range(bn // wn // 16):
                    inside("W fragment", bm * 128 + (wc * (bn // wn) + lr) * 128 + f * 2048 + ch, 16, bm * 128 + bn * 128)
            for f in range(bm // wm // 16):
                inside("A scale", bm * 128 + bn * 128 + (wr * (bm // wm) + lr) * 8 + g * 2 + f * 128, 2, stage)
            for f in range(bn // wn // 16):
                inside("W scale", bm * 128 + bn * 128 + (bm + wc * (bn // wn) + lr) * 8 + g * 2 + f * 128, 2, stage)
    if kg == 2:
        assert waves * (bm // (16 * wm)) * (bn // (16 * wn)) * 64 * 16 <= lds
    # results: columns in fours (N % 8 == 0), rows below M; partial sums [split][batch][M][N]
    tk = bm // (16 * wm) // kg
    for tm, tn in tiles:
        for wave in range(waves):
            wr, wc = wave // wn, wave % wn
            for k in range(kg):
                m = tm * bm + wr * (bm // wm) + (k * tk * 16 if kg == 2 else 0) + np.arange(tk)[:, None, None] * 16 + lr[None, None, :]
                n0 = tn * bn + wc * (bn // wn) + g[None, None, :] * 4 + np.arange(bn // wn // 16)[None, :, None] * 16
                ok = (m < M) & (n0 < N)
                m_, n_ = np.broadcast_to(m, ok.shape)[ok], np.broadcast_to(n0, ok.shape)[ok]
                inside("C", m_ * N + n_, 4, M * N)
                inside("partial sums", ((splits - 1) * batch + batch - 1) * M * N + m_ * N + n_, 4, splits * batch * M * N)


@pytest.mark.parametrize("seed", range(5))
def test_product(seed):
    rng = random.Random(seed)
    taken = set()
    sizes = [_product_sizes(rng) for _ in range(25)] + [(1, 500, 3200, 1100), (1, 900, 4000, 700), (1, 1900, 4072, 264), (1, 70, 136, 13000), (1, 4300, 64, 300)]
    for batch, M, N, K in sizes:
        n = mx_plan(batch, M, N, K, True, False)
        if n["cfg"] < 0:
            _skinny(batch, M, N, K)
        else:
            _tile(batch, M, N, K, n["cfg"], n["splits"])
        taken.add((n["cfg"], n["splits"] > 1))
    assert taken >= {(-1, False), (0, False), (1, False), (2, False), (3, False), (3, True)}


# ---- attention -------------------------------------------------------------------------------------------------------------------------
def attention_plan(B, Hq, Hkv, Sq, Sk, D, docs, causal):
    group = Hq // Hkv
    pack = min(group, 8)
    while group % pack:
        pack -= 1
    rows, sets = Sq * pack, B * (Hq // pack)
    few, key_tiles = rows <= 16, cdiv(Sk, 64)
    rt = 1 if sets * cdiv(rows, 128) <= (512 if causal and key_tiles >= 16 else 384 if D == 64 else 256) else 2
    row_tiles = 1 if few else cdiv(rows, 64 * rt)
    wgs = sets * row_tiles
    s = min(512 // wgs, (Sk + 255) // (256 if few else 512))
    s = 1 if s < 1 or (not few and wgs >= 192) else min(s, 256)
    return dict(group=group, pack=pack, few=few, rt=rt, row_tiles=row_tiles, key_tiles=key_tiles, splits=s,
                part=s * sets * rows * (D + 2) * 4 if s > 1 else 0, range=B * key_tiles * 8 if docs and not few else 0)


def swz(D, row):
    return 2 * ((row & 3) | ((row >> 3) & 1) << 2) if D == 128 else 2 * (((row >> 1) & 1) | ((row >> 3) & 1) << 1)


class Attention:
    """One geometry: tensors with their strides (elements) and extents."""

    def __init__(self, rng, B, Hq, Hkv, Sq, Sk, D, causal, ragged, reach, heads_last):
        self.B, self.Hq, self.Hkv, self.Sq, self.Sk, self.D, self.causal, self.reach = B, Hq, Hkv, Sq, Sk, D, causal, reach
        self.n = attention_plan(B, Hq, Hkv, Sq, Sk, D, 1, causal)
        self.q = (Sq * Hq * D, D, Hq * D) if heads_last else (Hq * Sq * D, Sq * D, D)
        self.kv = (Sk * Hkv * D, D, Hkv * D) if heads_last else (Hkv * Sk * D, Sk * D, D)
        self.first = [rng.choice([Sk - Sq, 0, rng.randint(-3, Sk + 3)]) for _ in range(B)]
        self.valid = [rng.choice([Sk, rng.randint(-1, Sk + 2)]) if ragged else Sk for _ in range(B)]
        self.prefix = [rng.randint(-1, Sk + 1) if ragged else 0 for _ in range(B)]

    def limit(self, b, qi):
        lim = min(self.valid[b], self.Sk)
        if self.causal:
            lim = min(lim, max(self.first[b] + qi + 1, self.prefix[b]))
        return max(lim, 0)

    def request(self, b, hk, key0, count, lds, lds_size):
        """A wave set's LDS-DMA of `count` rows from key0 on: what the resource lets through is inside the tensor."""
        D, (kb, kh, ks) = self.D, self.kv
        rows = min(count, self.Sk - key0)
        assert rows > 0
        extent = (rows - 1) * ks * 2 + 2 * D
        per = 64 // (D // 8)
        lane = np.arange(64)
        pieces = count // per
        base = (b * kb + hk * kh + key0 * ks) * 2
        total = self.B * self.Hkv * self.Sk * D * 2
        got = set()
        for piece in range(pieces):
            r = piece * per + lane // (D // 8)
            chunk = (lane % (D // 8)) ^ swz(D, r)
            # the kernels' form: the first piece's chunk, with bit 3 of the row flipped in where the piece's rows have it
            if count == 32:
                i = piece
                base_piece_row = lane // (D // 8)
            else:
                i = piece % (pieces // 4)
                base_piece_row = piece // (pieces // 4) * (pieces // 4) * per + lane // (D // 8)
            vc = (lane % (D // 8)) ^ swz(D, lane // (D // 8))
            flip = ((vc ^ swz(D, 8)) - vc) * 16
            off = base_piece_row * ks * 2 + vc * 16 + np.where((i * per) & 8, flip, 0) + i * per * ks * 2
            assert (off >= 0).all() and off.max() < 2 ** 31
            if (base_piece_row & 8).max() == 0:
                assert (off == r * ks * 2 + chunk * 16).all()
            through = off < extent
            inside("K / V", base + off[through], 16, total)
            inside("LDS", lds + piece * 1024 + lane * 16, 16, lds_size)
            got |= {int(x) for x in off[through]}
        # every byte of every row that exists arrives
        assert got >= {r * ks * 2 + c * 16 for r in range(rows) for c in range(D // 8)}

    def check(self):
        n, B, Hq, Sq, Sk, D = self.n, self.B, self.Hq, self.Sq, self.Sk, self.D
        pack, splits = n["pack"], n["splits"]
        nsets, rows = Hq // pack, Sq * pack
        trows = 16 if n["few"] else 64 * n["rt"]
        lane = np.arange(64)
        lr, lq = lane & 15, lane >> 4
        waves = 1 if n["few"] else 4
        oper = (32 if n["few"] else 64) * 2 * D
        win = 31 + Sq if n["few"] else 64 + (trows - 1) // pack + 2
        if n["few"]:
            lds = max(8 * oper + 4 * win * pack * 4, 3 * 16 * D * 4 + 3 * 2 * 64 * 4)
        else:
            lds = 4 * oper + 512 + 2 * win * pack * 4
        assert lds <= 160 * 1024 and pack * win <= (320 if n["few"] else 768)
        out_seen = 0
        for b in range(B):
            for set_ in {0, nsets - 1}:
                head0 = set_ * pack
                hk = head0 // n["group"]
                assert (head0 + pack - 1) // n["group"] == hk                # a packed set shares one K / V head
                for tile in {0, n["row_tiles"] - 1, n["row_tiles"] // 2}:
                    q_first, q_last = tile * trows // pack, min((tile * trows + trows - 1) // pack, Sq - 1)
                    if n["few"]:
                        q_first, q_last = 0, Sq - 1
                    assert 0 <= q_first <= q_last
                    row = tile * trows + np.arange(waves * (trows // waves if not n["few"] else 16))
                    qi = row // pack
                    live = qi < Sq
                    hg = np.where(live, row % pack, pack - 1)
                    qi = np.where(live, qi, Sq - 1)
                    for e in range(0, D, 8):
                        inside("q", b * self.q[0] + (head0 + hg) * self.q[1] + qi * self.q[2] + e, 8, B * Hq * Sq * D)
                    back = hg * win + (q_last - qi)
                    keys = 32 if n["few"] else 64
                    inside("bias window reads", back[live].reshape(-1, 1) + np.arange(keys)[None, :], 1, pack * win)
                    inside("bias window reads", back.reshape(-1, 1) + np.arange(keys)[None, :], 1, pack * win)
                    # bias fetches
                    for t in {0, cdiv(Sk, keys) - 1}:
                        at = np.minimum(np.arange(320 if n["few"] else 768), pack * win - 1)
                        g = at // win
                        frm = max(-0x40000000, min(0x40000000, t * keys - (self.first[b] + q_last)))
                        dist = np.clip(frm + at - g * win, -self.reach, self.reach)
                        inside("bias", (head0 + g) * (2 * self.reach + 1) + self.reach + dist, 1, Hq * (2 * self.reach + 1))
                    lim = self.limit(b, q_last)
                    assert all(self.limit(b, int(i)) <= lim for i in qi)     # the limit grows with the query
                    blocks = cdiv(lim, keys)
                    for split in {0, splits - 1}:
                        b0, b1 = blocks * split // splits, blocks * (split + 1) // splits
                        assert 0 <= b0 <= b1 <= cdiv(Sk, keys)
                        for t in {b0, b1 - 1} if b1 > b0 else ():
                            self.request(b, hk, t * keys, keys, 0, oper)
                            if n["few"]:
                                key = np.minimum(t * 32 + 8 * (lr >> 2) + 4 * np.arange(2)[:, None] + (lr & 3), Sk - 1)
                                for s in range(D // 32):
                                    inside("K", b * self.kv[0] + hk * self.kv[1] + key * self.kv[2] + (s * 4 + lq) * 8, 8, B * self.Hkv * Sk * D)
                    # results and partial results
                    inn, qs = row[live], qi[live]
                    for d in range(D // 16):
                        for q4 in range(4):
                            inside("out", b * Sq * Hq * D + qs * Hq * D + (head0 + inn % pack) * D + q4 * 4 + d * 16, 4, B * Sq * Hq * D)
                    if splits > 1:
                        part_row = (splits - 1) * B * nsets * rows + (b * nsets + set_) * rows + inn
                        inside("partial rows", part_row * D, D, n["part"] // 4)
                        inside("maximum, sum", splits * B * nsets * rows * D + part_row * 2, 2, n["part"] // 4)
                    out_seen += 1
        if splits > 1:
            assert B * nsets * rows == B * Hq * Sq                            # the joins' rows
            row = np.unique(np.linspace(0, B * Hq * Sq - 1, 50).astype(I))
            set_all = row // rows
            inn = row - set_all * rows
            inside("joined out", set_all // nsets * Sq * Hq * D + inn // pack * Hq * D + (set_all % nsets * pack + inn % pack) * D, D, B * Sq * Hq * D)
        # LDS reads of fragments: a block is 32 rows
        for at in range(0, oper, 64 * D):
            krow = 8 * ((lane & 15) >> 2) + (lane & 3)
            klane = krow * 2 * D + (((lane >> 4) ^ swz(D, krow)) << 4)
            for s in range(D // 32):
                for kt in range(2):
                    inside("K fragment", ((at + klane) ^ (s * 64)) + kt * 8 * D, 16, oper)
            vrow = 8 * (lane >> 4) + ((lane & 15) >> 2)
            vlane = vrow * 2 * D + ((((lane & 3) >> 1) ^ swz(D, vrow)) << 4) + (lane & 1) * 8
            for d in range(D // 16):
                for half in (0, 8 * D):
                    inside("V fragment", ((at + vlane) ^ (d * 32)) + half, 8, oper)
        assert out_seen


@pytest.mark.parametrize("seed", range(8))
def test_attention(seed):
    rng = random.Random(seed)
    kinds = set()
    for k in range(40):
        Hkv, group, D = rng.choice([1, 2, 4]), rng.choice([1, 2, 3, 4, 7, 9, 11, 16]), rng.choice([64, 128])
        Sq = rng.choice([1, 1, 2, 5, rng.randint(1, 40), rng.randint(40, 700)])
        Sk = rng.choice([rng.randint(1, 70), rng.randint(1, 900), rng.randint(900, 9000)])
        if k % 8 == 0:
            Hkv, group, Sq, Sk = 8, 16, 900, 100                              # 128-row tiles
        a = Attention(rng, rng.randint(1, 3), Hkv * group, Hkv, Sq, Sk, D, rng.random() < 0.6, rng.random() < 0.5, rng.choice([0, 1, 32, 1000]),
                      rng.random() < 0.5)
        a.check()
        kinds.add((a.n["few"], a.n["rt"], a.n["splits"] > 1))
    assert {f for f, _, _ in kinds} == {True, False} and {r for f, r, _ in kinds if not f} == {1, 2} and {s for _, _, s in kinds} == {True, False}


def test_requests_stay_in_32_bits():
    """The greatest row stride that is taken (below 2^24 elements): a tile's offsets and its resource's extent."""
    step = (1 << 24) - 8
    for D in (64, 128):
        assert 63 * step * 2 + 2 * D < 2 ** 31

"""Generates easyanimate_amd/csrc/ea_gemm_mxfp4_w4_loop.inc: the hand-placed main loop of gemm256_mxfp4_w4_kernel as ONE inline-asm
block -- the loop of gen_gemm_w4_asm.py (same tiles in bytes, same fragment buffers, same rules for the placement, same hand-overs: see there) on
v_mfma_scale_f32_16x16x128_f8f6f4, with the scales added:

    python tools/gen_gemm_mxfp4_asm.py            (rewrites the .inc)

  * a K tile's 2 x 2 KiB of scale bytes are one more LDS-DMA request per wave (waves 0, 1: activation rows, 2, 3: weight rows), in front
    of the tile's W requests; two stages of 4 KiB behind the operand stages;
  * the lane's 8 + 8 scale pairs of tile t + 1 (u16: the byte of k-step 0, the byte of k-step 1) are read into the register set that tile
    t does not use, behind the barrier that says W(t + 1) -- and with it the older scale request -- has landed;
  * the two sets alternate, so the loop body is two tiles long."""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import gen_gemm_w4_asm as g      # noqa: E402

OUT = os.environ.get("EA_GEN_OUT") or os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "easyanimate_amd", "csrc", "ea_gemm_mxfp4_w4_loop.inc")

SCALE = [196, 212]                # first VGPR of scale set b: 8 weight pairs, 8 activation pairs
V_SW, V_SA = 228, 229             # LDS byte addresses of the scale reads, toggled by xor 0x1000
S_RS, S_KS, S_NRS, S_KSTS, S_MS = 72, 76, 77, 78, 79      # resource (4 SGPRs), offset of the requested tile, num_records, K step, LDS address


def mfma(b, n, p, zero_c=False):
    """MFMA n of k-step b with scale set p: the weight fragment is the A operand (C^T orientation)."""
    j, i = n >> 3, n & 7
    a = g.acc(i, j)
    w, x = f"v[{g.FW[b] + 4 * j}:{g.FW[b] + 4 * j + 3}]", f"v[{g.FA[b] + 4 * i}:{g.FA[b] + 4 * i + 3}]"
    c = "0" if zero_c else f"a[{a}:{a + 3}]"
    return (f"v_mfma_scale_f32_16x16x128_f8f6f4 a[{a}:{a + 3}], {w}, {x}, {c}, v{SCALE[p] + j}, v{SCALE[p] + 8 + i} "
            f"op_sel:[{b},{b},0] op_sel_hi:[0,0,0] cbsz:4 blgp:4")


def rd_scale(f, p):
    """Scale pair f (0..7 weight, 8..15 activation) into set p."""
    off = f" offset:{(f & 7) * 128}" if f & 7 else ""
    return f"ds_read_u16 v{SCALE[p] + f}, v{V_SW if f < 8 else V_SA}{off}"


def dma_scale():
    return f"buffer_load_dwordx4 %[soff], s[{S_RS}:{S_RS + 3}], s{S_KS} offen lds"


def schedule(p):
    """The base schedule plus the scales; p = scale set of this tile (the next tile's pairs go to p ^ 1)."""
    s = g.schedule()

    def free(n):
        while s[n]:
            n += 1
        return n
    # the scale request in front of the W requests, between the barrier that frees their stage and the first of them
    n = g.REQUEST_W - 1
    assert s[n][-1] == g.m0_first("w") and g.FREE_W < n
    s[g.FREE_W].append(f"s_mov_b32 m0, s{S_MS}")
    s[n].insert(-1, dma_scale())
    n = g.FREE_A + 1
    for v in (V_SW, V_SA):
        n = free(n)
        s[n].append(f"v_xor_b32 v{v}, 0x1000, v{v}")
    n = g.READ_W0
    for f in range(16):
        n = free(n)
        s[n].append(rd_scale(f, p ^ 1))
    n = g.REQUEST_A + 7 * g.REQUEST_STEP + 1
    for ins in (f"s_add_u32 s{S_KS}, s{S_KS}, s{S_KSTS}", f"s_xor_b32 s{S_MS}, s{S_MS}, 0x1000"):
        n = free(n)
        s[n].append(ins)
    s = g.finish(s)
    # no scale register of the set in use is written before its last MFMA; scale reads end where the fragment reads do
    for n in s:
        for i in s[n]:
            if i.startswith("ds_read_u16"):
                r = int(i.split()[1].strip("v,"))
                assert SCALE[p ^ 1] <= r < SCALE[p ^ 1] + 16 and g.LANDED_W < n <= 128 - g.LATENCY
    return s


def loop_body():
    base = g.loop_body(g.finish(g.schedule()), False, True)
    body = []
    B = body.append
    # ---- the base prologue up to its first K tile, with the scale resource, addresses, requests and first reads put in
    end = next(k for k, i in enumerate(base) if i.startswith("s_cmp_gt_u32") and i.endswith(", 2"))
    pro = base[:end]
    w0 = g.m0_first("w")
    tiles = 0
    for k, ins in enumerate(pro):
        if ins == w0:                                 # in front of a tile's W requests: its scale request
            if tiles == 1:                            # tile 1 -> stage 1
                B(f"s_cmp_gt_u32 s{g.S_LEFT}, 1")
                B(f"s_cselect_b32 s{S_RS + 2}, s{S_NRS}, 0")
                B(f"s_mov_b32 s{S_KS}, s{S_KSTS}")
                B(f"s_xor_b32 s{S_MS}, s{S_MS}, 0x1000")
            B(f"s_mov_b32 m0, s{S_MS}")
            B("s_nop 0")
            B(dma_scale())
            tiles += 1
        if ins.startswith("s_waitcnt vmcnt("):        # tile 0 has landed: tile 1's 17 requests and the 16 bias / gate loads may be left
            assert ins == "s_waitcnt vmcnt(32)"
            ins = "s_waitcnt vmcnt(33)"
        B(ins)
        if k == 0:
            for r, v in ((S_RS, "s_lo"), (S_RS + 1, "s_hi"), (S_RS + 2, "s_ext"), (S_NRS, "s_ext"), (S_KSTS, "s_kst"), (S_MS, "lds_s")):
                B(f"s_mov_b32 s{r}, %[{v}]")
            B(f"s_mov_b32 s{S_RS + 3}, 0x00020000")
            B(f"s_mov_b32 s{S_KS}, 0")
            B(f"v_mov_b32 v{V_SW}, %[sw0]")
            B(f"v_mov_b32 v{V_SA}, %[sa0]")
    assert tiles == 2
    B(f"s_xor_b32 s{S_MS}, s{S_MS}, 0x1000")          # the loop's first request (tile 2) goes to stage 0 again
    B(f"s_add_u32 s{S_KS}, s{S_KS}, s{S_KSTS}")
    for f in range(16):
        B(rd_scale(f, 0))

    def k_tile(p, first):
        s = schedule(p)
        B(f"s_cmp_gt_u32 s{g.S_LEFT}, 2")             # tile t + 2 exists?
        B(f"s_cselect_b32 s{g.S_RA + 2}, s{g.S_NRA}, 0")
        B(f"s_cselect_b32 s{g.S_RW + 2}, s{g.S_NRW}, 0")
        B(f"s_cselect_b32 s{S_RS + 2}, s{S_NRS}, 0")
        B("s_waitcnt lgkmcnt(0)")                     # fragment buffer 0 and the scales of this tile
        for n in range(128):
            for ins in s[n]:
                if first and ins.startswith("s_waitcnt vmcnt("):       # the bias / gate loads are younger than tile 1's requests
                    ins = f"s_waitcnt vmcnt({int(ins[len('s_waitcnt vmcnt('):-1]) + 16})"
                B(ins)
            B(mfma(0 if n < 64 else 1, n & 63, p, zero_c=first and n < 64))
        for ins in s[128]:
            B(ins)

    k_tile(0, True)
    B(f"s_cmp_lg_u32 s{g.S_LEFT}, 0")
    B("s_cbranch_scc0 9f")                            # nk == 1
    B("1:")
    k_tile(1, False)
    B(f"s_cmp_lg_u32 s{g.S_LEFT}, 0")
    B("s_cbranch_scc0 9f")
    k_tile(0, False)
    B(f"s_cmp_lg_u32 s{g.S_LEFT}, 0")
    B("s_cbranch_scc1 1b")
    B("9:")
    # everything this wave requested has landed, the last MFMAs have left the pipe
    B("s_waitcnt vmcnt(0) lgkmcnt(0)")
    B("s_nop 15")
    B("s_nop 15")
    return body


def emit():
    L = ["// GENERATED by tools/gen_gemm_mxfp4_asm.py -- do not edit; see that file for the schedule.", "#define EA_MXW4_MAINLOOP_ASM \\"]
    body = loop_body()
    L += [f'    "{ins}\\n\\t" \\' for ins in body]
    L[-1] = L[-1][:-2]
    L.append("")
    clob = [f'"v{r}"' for r in list(range(132)) + list(range(SCALE[0], V_SA + 1))] + [f'"s{r}"' for r in range(S_RS, 102)] + ['"m0"', '"scc"', '"memory"']
    L.append("#define EA_MXW4_CLOBBERS \\")
    for k in range(0, len(clob), 16):
        L.append("    " + ", ".join(clob[k:k + 16]) + (", \\" if k + 16 < len(clob) else ""))
    L.append("")
    open(OUT, "w").write("\n".join(L))
    print(OUT, len(body), "asm lines")


if __name__ == "__main__":
    emit()

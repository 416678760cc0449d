"""CPU: the range coder chain's generated loop (genozip_amd/csrc/gz_chain_asm.h), which only the GPU executes, instruction by instruction
in an interpreter of the few instructions it is made of - 64 lanes, the exec mask, double precision with truncation in exact integers -
against the integer recurrence of the coder: every checkpoint at its address and nothing else written, the final state, every access
inside its buffer. The interpreter refuses what the hardware does not interlock: a DPP read of a register that a vector instruction
wrote less than two wait states before, a read of a register whose load has not been waited for, an end of the loop with a store in flight."""
import os
import random
import re
import struct

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HDR = os.path.join(ROOT, "genozip_amd", "csrc", "gz_chain_asm.h")
M32, M64 = (1 << 32) - 1, (1 << 64) - 1
NAN = 0x7ff8000000000000


def fma_rtz(a, b, c):
    """fma of three doubles given as bits, truncated; what is not finite, or too small for a normal number, is no case of the coder's: NaN, 0"""
    def dec(x):
        e = (x >> 52) & 0x7ff
        if e == 0x7ff:
            return None
        m = (x & ((1 << 52) - 1)) | ((1 << 52) if e else 0)
        return (-m if x >> 63 else m), (e or 1) - 1075
    da, db, dc = dec(a), dec(b), dec(c)
    if da is None or db is None or dc is None:
        return NAN
    (ma, ea), (mb, eb), (mc, ec) = da, db, dc
    m, e = ma * mb, ea + eb
    if not m:
        m, e = mc, ec
    elif mc:
        if e > ec:
            m, e = (m << (e - ec)) + mc, ec
        else:
            m += mc << (ec - e)
    if not m:
        return 0
    s, m = (1, -m) if m < 0 else (0, m)
    sh = m.bit_length() - 53
    m, e = (m >> sh if sh > 0 else m << -sh), e + sh
    be = e + 1075
    if be >= 0x7ff:
        return NAN
    if be <= 0:
        return 0
    return s << 63 | be << 52 | (m & ((1 << 52) - 1))


def f64(x):
    return struct.unpack("<Q", struct.pack("<d", x))[0]


class Wave:
    def __init__(self, lines, env, mem_r, base_r, mem_w, base_w):
        self.L, self.env = lines, env
        self.mem_r, self.base_r, self.mem_w, self.base_w = mem_r, base_r, mem_w, base_w
        self.V = [[0xdeadbeef ^ (r * 2654435761 & M32)] * 64 for r in range(256)]
        self.S = [0xabad1dea] * 104
        self.exec, self.scc, self.slot = M64, 0, 0
        self.wrote = [-10] * 256          # issue slot in which a vector instruction wrote the register
        self.loading = set()
        self.stores = 0
        self.written = set()

    # -- operands
    def reg(self, t):
        m = re.fullmatch(r"([vs])\[(\d+):(\d+)\]", t) or re.fullmatch(r"([vs])(\d+)", t)
        assert m, t
        return m.group(1), int(m.group(2))

    def rv(self, r):
        assert r not in self.loading, "v%d is read before its load was waited for" % r
        return self.V[r]

    def src32(self, t):
        if re.fullmatch(r"-?(0x[0-9a-f]+|\d+)", t):
            return [int(t, 0) & M32] * 64
        k, n = self.reg(t)
        return self.rv(n) if k == "v" else [self.S[n]] * 64

    def src64(self, t):
        neg = t.startswith("-v")
        t = t[1:] if neg else t
        if t == "1.0":
            return [f64(1.0)] * 64
        k, n = self.reg(t)
        assert k == "v"
        return [(lo | hi << 32) ^ (neg << 63) for lo, hi in zip(self.rv(n), self.rv(n + 1))]

    def set32(self, r, vals):
        assert r not in self.loading, "v%d is written with a load to it in flight" % r
        if self.exec == M64:
            self.V[r] = list(vals)
        else:
            self.V[r] = [v if self.exec >> i & 1 else o for i, (v, o) in enumerate(zip(vals, self.V[r]))]
        self.wrote[r] = self.slot

    def set64(self, r, vals):
        self.set32(r, [v & M32 for v in vals])
        self.set32(r + 1, [v >> 32 for v in vals])

    def s64(self, t):
        if t == "exec":
            return self.exec
        if t in ("1", "-1"):
            return int(t) & M64
        k, n = self.reg(t)
        assert k == "s"
        return self.S[n] | self.S[n + 1] << 32

    def dpp_ready(self, r):
        assert self.slot - self.wrote[r] > 2, "DPP read of v%d %d slots after its write" % (r, self.slot - self.wrote[r])

    # -- run
    def run(self):
        labels, ins = {}, []
        for ln in self.L:
            if ln.endswith(":"):
                labels[ln[:-1]] = len(ins)
            elif not ln.startswith("."):
                ins.append(ln)
        pc = 0
        while pc < len(ins):
            ln = ins[pc]
            for k, v in self.env.items():
                ln = ln.replace(k, v)
            op, _, rest = ln.partition(" ")
            mods = re.findall(r"\b(\w+):(0x\w+|\w+)", re.sub(r"[vs]\[\d+:\d+\]", "", rest))
            a = [t.strip() for t in re.sub(r"\s+(row_newbcast|wave_ror|row_mask|bank_mask|offset):\S+", "", rest).split(",")] if rest else []
            pc += 1
            self.slot += 1
            if op.startswith("v_"):
                assert self.exec == M64, "a vector instruction with lanes switched off: " + ln
            op0 = op.replace("_e64", "")
            if op0 == "s_nop":
                self.slot += int(a[0])
            elif op0 == "s_waitcnt":
                if "vmcnt(0)" in ln:
                    self.loading.clear()
                    self.stores = 0
            elif op0 == "s_mov_b32":
                self.S[self.reg(a[0])[1]] = self.src32(a[1])[0]
            elif op0 == "s_mov_b64":
                if a[0] == "exec":
                    self.exec = self.s64(a[1])
                else:
                    n, v = self.reg(a[0])[1], self.s64(a[1])
                    self.S[n], self.S[n + 1] = v & M32, v >> 32
            elif op0 == "s_lshl_b64":
                n, v = self.reg(a[0])[1], self.s64(a[1]) << int(a[2]) & M64
                self.S[n], self.S[n + 1], self.scc = v & M32, v >> 32, int(v != 0)
            elif op0 in ("s_add_u32", "s_addc_u32"):
                v = self.src32(a[1])[0] + self.src32(a[2])[0] + (self.scc if op0 == "s_addc_u32" else 0)
                self.S[self.reg(a[0])[1]], self.scc = v & M32, v >> 32
            elif op0 == "s_sub_u32":
                x, y = self.src32(a[1])[0], self.src32(a[2])[0]
                self.S[self.reg(a[0])[1]], self.scc = (x - y) & M32, int(y > x)
            elif op0 == "s_cmp_lt_u32":
                self.scc = int(self.src32(a[0])[0] < self.src32(a[1])[0])
            elif op0 == "s_cmp_eq_u32":
                self.scc = int(self.src32(a[0])[0] == self.src32(a[1])[0])
            elif op0 == "s_cselect_b32":
                self.S[self.reg(a[0])[1]] = self.src32(a[1] if self.scc else a[2])[0]
            elif op0 in ("s_branch", "s_cbranch_scc1"):
                if op0 == "s_branch" or self.scc:
                    pc = labels[a[0][:-1]]
            elif op0 == "v_mbcnt_lo_u32_b32":
                assert a[1] == "-1"
                self.set32(self.reg(a[0])[1], [min(i, 32) + v for i, v in enumerate(self.src32(a[2]))])
            elif op0 == "v_mbcnt_hi_u32_b32":
                assert a[1] == "-1"
                self.set32(self.reg(a[0])[1], [max(i - 32, 0) + v for i, v in enumerate(self.src32(a[2]))])
            elif op0 == "v_mov_b32":
                self.set32(self.reg(a[0])[1], self.src32(a[1]))
            elif op0 == "v_mov_b64":
                d, n = self.reg(a[0])[1], self.reg(a[1])[1]
                lo, hi = self.rv(n), self.rv(n + 1)
                self.set32(d, lo)
                self.set32(d + 1, hi)
            elif op0 == "v_add_u32":
                self.set32(self.reg(a[0])[1], [(x + y) & M32 for x, y in zip(self.src32(a[1]), self.src32(a[2]))])
            elif op0 == "v_mul_u32_u24":
                self.set32(self.reg(a[0])[1], [(x & 0xffffff) * (y & 0xffffff) & M32 for x, y in zip(self.src32(a[1]), self.src32(a[2]))])
            elif op0 == "v_lshlrev_b32":
                self.set32(self.reg(a[0])[1], [y << (x & 31) & M32 for x, y in zip(self.src32(a[1]), self.src32(a[2]))])
            elif op0 == "v_lshrrev_b32":
                self.set32(self.reg(a[0])[1], [y >> (x & 31) for x, y in zip(self.src32(a[1]), self.src32(a[2]))])
            elif op0 == "v_lshlrev_b64":
                self.set64(self.reg(a[0])[1], [y << int(a[1]) & M64 for y in self.src64(a[2])])
            elif op0 == "v_xor_b32":
                self.set32(self.reg(a[0])[1], [x ^ y for x, y in zip(self.src32(a[1]), self.src32(a[2]))])
            elif op0 == "v_and_or_b32":
                self.set32(self.reg(a[0])[1], [x & y | z for x, y, z in zip(*(self.src32(t) for t in a[1:4]))])
            elif op0 == "v_cndmask_b32":
                m = self.s64(a[3])
                self.set32(self.reg(a[0])[1], [y if m >> i & 1 else x for i, (x, y) in enumerate(zip(self.src32(a[1]), self.src32(a[2])))])
            elif op0 == "v_mov_b32_dpp":
                assert dict(mods) == {"wave_ror": "1", "row_mask": "0xf", "bank_mask": "0xf"}
                n = self.reg(a[1])[1]
                self.dpp_ready(n)
                s = self.rv(n)
                self.set32(self.reg(a[0])[1], [s[(i - 1) % 64] for i in range(64)])
            elif op0 == "v_fma_f64":
                self.set64(self.reg(a[0])[1], [fma_rtz(*t) for t in zip(*(self.src64(t) for t in a[1:4]))])
            elif op0 == "v_fmac_f64_dpp":
                md = dict(mods)
                assert md["row_mask"] == md["bank_mask"] == "0xf"
                n, lane = self.reg(a[1])[1], int(md["row_newbcast"])
                self.dpp_ready(n)
                self.dpp_ready(n + 1)
                s, f, d = self.src64(a[1]), self.src64(a[2]), self.src64(a[0])
                self.set64(self.reg(a[0])[1], [fma_rtz(s[i // 16 * 16 + lane], f[i], d[i]) for i in range(64)])
            elif op0 == "global_load_dwordx3":
                off = int(dict(mods).get("offset", "0"))
                assert self.exec == M64
                d, addr, base = self.reg(a[0])[1], self.src32(a[1]), self.s64(a[2])
                at = [base + x + off - self.base_r for x in addr]
                assert min(at) >= 0 and max(at) + 12 <= len(self.mem_r)
                for k in range(3):
                    self.set32(d + k, [struct.unpack_from("<I", self.mem_r, p + 4 * k)[0] for p in at])
                self.loading.update(range(d, d + 3))
            elif op0 == "global_store_dwordx2":
                addr, n, base = self.src32(a[0]), self.reg(a[1])[1], self.s64(a[2])
                lo, hi = self.rv(n), self.rv(n + 1)
                for i in range(64):
                    if self.exec >> i & 1:
                        p = base + addr[i] - self.base_w
                        assert 0 <= p and p + 8 <= len(self.mem_w) and p % 8 == 0
                        struct.pack_into("<II", self.mem_w, p, lo[i], hi[i])
                        assert p not in self.written
                        self.written.add(p)
                self.stores += 1
            else:
                raise AssertionError("an instruction the interpreter does not know: " + ln)
        assert not self.stores and not self.loading and self.exec == M64


def header():
    src = open(HDR).read()
    block = int(re.search(r"#define GZ_CHAIN_BLOCK (\d+)", src).group(1))
    assert re.search(r"#define GZ_CHAIN_REC 12\b", src)
    return block, re.findall(r'^\s+"(.*)\\n\\t" \\$', src, re.M), src


@pytest.mark.parametrize("nblk", [1, 2, 3])
def test_chain_loop_in_an_interpreter(nblk):
    block, lines, src = header()
    rnd = random.Random(nblk)
    n = nblk * block
    recs, states = bytearray(), []
    rng = 0xffffffff
    for i in range(n):                                   # totals small and large, symbols rare and frequent: 0, 1 and 2 bytes out
        tot = rnd.choice([1, 2, rnd.randrange(1, 300), rnd.randrange(1, 65520), 65519])
        freq = rnd.choice([1, tot, rnd.randrange(1, tot + 1)])
        states.append(rng)
        rng = (rng // tot) * freq
        while rng < 1 << 24:
            rng = rng << 8
        inv = f64(2.0 ** -45 / tot)                      # rounded up to a multiple of 2^16 units; the symbol's cum in those bits
        inv = (inv + 0xffff & ~0xffff) | rnd.choice([0, 0xffff, rnd.randrange(1 << 16)])
        recs += struct.pack("<III", inv & M32, inv >> 32, f64(freq * 2.0 ** 45) >> 32)
    ck = bytearray(8 * (n // 64))
    base_r, base_w = 0x7ffff000, 0x1fffffff0             # (both bases carry into the high word on the way)
    env = {"%[rlo]": "v0", "%[rhi]": "v1", "%[blo]": "s0", "%[bhi]": "s1", "%[nblk]": "s2", "%[clo]": "s3", "%[chi]": "s4"}
    w = Wave(lines, env, bytes(recs), base_r, ck, base_w)
    first = f64(states[0] / 128.0)
    w.V[0], w.V[1] = [first & M32] * 64, [first >> 32] * 64
    w.S[0], w.S[1], w.S[2], w.S[3], w.S[4] = base_r & M32, base_r >> 32, nblk, base_w & M32, base_w >> 32
    before_v, before_s = [list(v) for v in w.V], list(w.S)
    w.run()
    assert len(w.written) == n // 64
    for c in range(n // 64):
        got = struct.unpack_from("<d", ck, 8 * c)[0]
        assert got * 128.0 == states[64 * c], c
    assert struct.unpack("<d", struct.pack("<II", w.V[0][0], w.V[1][0]))[0] * 128.0 == rng
    # nothing outside the clobber list was touched
    clob = re.search(r"#define GZ_CHAIN_F64_CLOBBERS (.*)", src).group(1)
    for r in range(2, 256):
        assert '"v%d"' % r in clob or w.V[r] == before_v[r], r
    for r in range(104):
        assert '"s%d"' % r in clob or w.S[r] == before_s[r], r


def test_nothing_writes_through_the_scalar_data_cache():
    """that cache is not coherent with the vector stores and loads of other kernels, and the range coder's chain publishes its checkpoints
    while the kernels that read them are already queued: no source compiled for the GPU holds a scalar store or atomic, a write-back or a discard"""
    bad = re.compile(r"\bs_" + r"(scratch_|buffer_)?" + r"(store|atomic)_" + r"|\bs_dcache_" + r"(wb|discard)")
    seen = 0
    for top in ("genozip_amd", "tools", "tests", "include", "oracle"):
        for d, _, files in os.walk(os.path.join(ROOT, top)):
            for f in files:
                if f.endswith((".h", ".hip", ".cpp", ".c", ".py", ".sh")):
                    seen += 1
                    text = open(os.path.join(d, f), errors="replace").read()
                    assert not bad.search(text), os.path.join(d, f)
    assert seen > 50


def test_inline_asm_holds_no_load_that_outlives_it():
    """the compiler takes an asm block's output registers as written at once and as free when unused: a load still in flight at the end of the block
    would write over whatever lives there by then. Every block with a load in it waits for it in the same block"""
    csrc = os.path.join(ROOT, "genozip_amd", "csrc")
    blocks = 0
    for f in sorted(os.listdir(csrc)):
        text = open(os.path.join(csrc, f)).read()
        for m in re.finditer(r"\basm\s*(?:volatile\s*)?\(", text):
            body = text[m.end():text.index(";", m.end())]
            if "GZ_CHAIN_F64_ASM" in body:
                continue                                     # (the loop: the interpreter above sees its loads home)
            blocks += 1
            if re.search(r"_load_|_read_|s_memtime|s_load", body):
                assert "s_waitcnt" in body.split("load")[-1], (f, body)
    assert blocks >= 3

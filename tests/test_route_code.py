"""The addresses of the router's global accesses, followed through the code the compiler makes of it: no GPU.

One wave is walked through the gfx950 code with its scalar registers and 64 lanes of vector registers.  What an instruction outside the few that
form addresses writes is unknown, what the compiler calls undefined is so too; at a branch on something unknown a walk takes either side.  Every
logit and every bias has to be read once, from a known address; ids and weights of the wave's token have to be all that is written."""
import os
import random
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cyb_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ALL, M32, M64 = (1 << 64) - 1, (1 << 32) - 1, (1 << 64) - 1
LOGITS, BIAS, IDS, WEIGHTS = (i << 36 for i in (1, 2, 3, 4))


def _signed(v):
    return v - (1 << 32) if v >> 31 else v


SCALAR = {"add_i32": lambda x, y: x + y, "sub_i32": lambda x, y: x - y, "mul_i32": lambda x, y: x * y,
          "mul_hi_u32": lambda x, y: x * y >> 32, "mul_hi_i32": lambda x, y: _signed(x) * _signed(y) >> 32,
          "lshl_b32": lambda x, y: x << (y & 31), "lshl_b64": lambda x, y: x << (y & 63), "ashr_i32": lambda x, y: _signed(x) >> (y & 31),
          "bfe_u32": lambda x, y: x >> (y & 31) & (1 << (y >> 16 & 127)) - 1,
          "and_b64": lambda x, y: x & y, "or_b64": lambda x, y: x | y, "andn2_b64": lambda x, y: x & ~y, "xor_b64": lambda x, y: x ^ y,
          "and_b32": lambda x, y: x & y, "or_b32": lambda x, y: x | y}
VECTOR = {"and_b32": lambda x, y: x & y, "or_b32": lambda x, y: x | y, "xor_b32": lambda x, y: x ^ y, "add_u32": lambda x, y: x + y,
          "sub_u32": lambda x, y: x - y, "subrev_u32": lambda x, y: y - x, "lshlrev_b32": lambda x, y: y << (x & 31),
          "lshrrev_b32": lambda x, y: y >> (x & 31), "lshlrev_b64": lambda x, y: y << (x & 63)}
VECTOR3 = {"lshl_add_u64": lambda x, y, z: (x << y) + z, "lshl_add_u32": lambda x, y, z: (x << y) + z, "lshl_or_b32": lambda x, y, z: x << y | z}
COMPARE = {"eq": lambda x, y: x == y, "ne": lambda x, y: x != y, "lg": lambda x, y: x != y, "lt": lambda x, y: x < y, "le": lambda x, y: x <= y,
           "gt": lambda x, y: x > y, "ge": lambda x, y: x >= y}


def _known(f, *values):
    return None if None in values else f(*values)


def _operands(rest):
    return [t.strip() for t in re.split(r",(?![^\[]*\])", rest)] if rest else []


def _registers(t):
    m = re.match(r"([sv])(?:(\d+)|\[(\d+):(\d+)\])$", t)
    if not m:
        return None
    first = int(m[2] or m[3])
    return m[1], range(first, int(m[4] or first) + 1)


class Code:
    """A kernel's instructions: (name, operands), labels by name, and where its arguments lie."""

    def __init__(self, body, kd, meta):
        self.code, self.labels = [], {}
        for line in body.split("\n"):
            undefined = re.findall(r"implicit-def: \$(\S+)", line)
            s = line.split(";")[0].strip()
            m = re.match(r"(\.LBB\w+):", s)
            if m:
                self.labels[m[1]] = len(self.code)
            elif undefined:
                self.code.append(("undefined", re.findall(r"([sv])gpr(\d+)", undefined[0])))
            elif s and not s.startswith("."):
                op, _, rest = s.partition(" ")
                self.code.append((re.sub(r"_e(32|64)$", "", op), _operands(rest)))
        self.group_size = int(re.search(r"\.offset:\s+(\d+)\s+\.size:\s+2\s+\.value_kind:\s+hidden_group_size_x", meta)[1])
        # scalar registers that a wave starts with: the arguments' address, the first arguments, then the workgroup's number.  The code of machines
        # that load arguments ahead begins behind the first branch.
        self.user = int(re.search(r"\.amdhsa_user_sgpr_count (\d+)", kd)[1])
        self.entry = self.labels[next(a[0] for op, a in self.code if op == "s_branch")]


class Wave:
    def __init__(self, code, args, block, rng):
        self.c, self.args, self.rng = code, args, rng
        self.s = {2 + i: args.get(4 * i) for i in range(code.user - 2)}
        self.s.update({0: 0, 1: 0, code.user: block})
        self.v = {0: list(range(64))}
        self.flag = {"scc": None, "vcc": None, "exec": ALL}
        self.sure = True                                             # (else: these lanes at most, any of them may be off)
        self.accesses = []

    def scalar(self, t):
        if t in ("vcc", "exec"):
            return self.flag[t]
        r = _registers(t)
        if r:
            return _known(lambda *w: sum(x << 32 * i for i, x in enumerate(w)), *(self.s.get(i) for i in r[1])) if r[0] == "s" else None
        try:
            return int(t, 0)
        except ValueError:
            return None

    def lanes(self, t):
        r = _registers(t)
        if r and r[0] == "v":
            parts = [self.v.get(i, [None] * 64) for i in r[1]]
            return [_known(lambda *w: sum(x << 32 * i for i, x in enumerate(w)), *w) for w in zip(*parts)]
        v = self.scalar(t)
        return [_known(lambda x: x & M64, v)] * 64

    def put(self, t, value):
        """One value for a scalar, 64 for a vector destination."""
        if t in ("vcc", "exec"):
            self.flag[t] = value
            return
        kind, regs = _registers(t)
        for i, r in enumerate(regs):
            if kind == "s":
                self.s[r] = _known(lambda x: x >> 32 * i & M32, value)
            else:
                old = self.v.get(r, [None] * 64)
                self.v[r] = [_known(lambda x: x >> 32 * i & M32, value[n]) if self.flag["exec"] >> n & 1 else old[n] for n in range(64)]

    def forget(self, op, a):
        for t in a[:2] if op.startswith(("v_div_scale", "v_permlane", "v_swap", "v_add_co", "v_mad_u64")) else a[:1]:
            if t == "vcc" or (_registers(t) or "x")[0] == "s":
                self.put(t, None)
            elif _registers(t):
                self.put(t, [None] * 64)
        if op.startswith("s_"):
            self.flag["scc"] = None

    def walk(self, limit=200000):
        pc = self.c.entry
        for _ in range(limit):
            op, a = self.c.code[pc]
            pc += 1
            if op == "s_endpgm":
                return self.accesses
            if op == "s_branch":
                pc = self.c.labels[a[0]]
            elif op.startswith("s_cbranch_"):
                cond = op[len("s_cbranch_"):]
                v = self.flag[cond[:3]] if cond.startswith(("scc", "vcc")) else self.flag["exec"] if self.sure or not self.flag["exec"] else None
                hit = self.rng.random() < 0.5 if v is None else bool(v) == (cond in ("scc1", "vccnz", "execnz"))
                if hit:
                    pc = self.c.labels[a[0]]
            else:
                self.step(op, a)
        raise AssertionError("a walk without an end")

    def step(self, op, a):
        name = op.partition("_")[2]
        if op in ("s_waitcnt", "s_nop", "s_barrier") or op.startswith(("ds_write", "s_setprio")):
            return
        if op == "undefined":
            for kind, r in a:
                (self.s if kind == "s" else self.v)[int(r)] = None if kind == "s" else [None] * 64
        elif op.startswith("s_load_dword"):
            for i, r in enumerate(_registers(a[0])[1]):
                self.s[r] = self.args.get(int(a[2], 0) + 4 * i)
        elif op.startswith(("global_", "flat_", "scratch_", "buffer_")):
            assert op.startswith(("global_load_", "global_store_")), op
            store = "store" in op
            at, base = (a[0], a[2]) if store else (a[1], a[2])
            more = re.search(r"offset:(-?\d+)", base)
            base = base.split()[0]
            origin = 0 if base == "off" else self.scalar(base)
            where = self.lanes(at)
            active = [n for n in range(64) if self.flag["exec"] >> n & 1]
            self.accesses.append((store, [_known(lambda x, b: x + b + int(more[1] if more else 0), where[n], origin) for n in active]))
            if not store:
                self.put(a[0], [None] * 64)
        elif op.startswith("s_cmp_"):
            x, y = (_known(lambda v: v & M32, self.scalar(t)) for t in a)
            if op.endswith("_i32"):
                x, y = (_known(_signed, v) for v in (x, y))
            self.flag["scc"] = _known(COMPARE[op[6:8]], x, y)
        elif op in ("s_mov_b32", "s_mov_b64"):
            self.put(a[0], _known(lambda x: x & M64, self.scalar(a[1])))
        elif op in ("s_cselect_b32", "s_cselect_b64"):
            scc = self.flag["scc"]
            self.put(a[0], None if scc is None else _known(lambda x: x & M64, self.scalar(a[1] if scc else a[2])))
        elif op == "s_and_saveexec_b64":
            old, v = self.flag["exec"], self.scalar(a[1])
            self.put(a[0], old)
            self.flag["exec"], self.sure = old if v is None else old & v, v is not None
            self.flag["scc"] = None if v is None else self.flag["exec"] != 0
        elif op in ("s_add_u32", "s_addc_u32"):
            v = _known(lambda x, y, c: (x & M32) + (y & M32) + c, self.scalar(a[1]), self.scalar(a[2]), 0 if op == "s_add_u32" else self.flag["scc"])
            self.put(a[0], _known(lambda x: x & M32, v))
            self.flag["scc"] = _known(lambda x: x >> 32, v)
        elif op.startswith("s_") and name in SCALAR:
            v = _known(SCALAR[name], _known(lambda x: x & M64, self.scalar(a[1])), _known(lambda x: x & M64, self.scalar(a[2])))
            v = _known(lambda x: x & (M64 if op.endswith("64") else M32), v)
            if a[0] == "exec":
                self.sure = v is not None
                v = self.flag["exec"] if v is None else v
            self.put(a[0], v)
            self.flag["scc"] = None if "add" in op or "sub" in op else _known(lambda x: x != 0, v)
        elif op == "v_readfirstlane_b32":
            self.put(a[0], self.lanes(a[1])[(self.flag["exec"] & -self.flag["exec"]).bit_length() - 1])
        elif op in ("v_mov_b32", "v_mov_b64"):
            self.put(a[0], self.lanes(a[1]))
        elif op.startswith("v_") and name in VECTOR and len(a) == 3:
            self.put(a[0], [_known(VECTOR[name], x, y) for x, y in zip(self.lanes(a[1]), self.lanes(a[2]))])
        elif op.startswith("v_") and name in VECTOR3:
            self.put(a[0], [_known(VECTOR3[name], *w) for w in zip(*(self.lanes(t) for t in a[1:4]))])
        elif op == "v_mad_u64_u32":
            self.put(a[1], None)
            self.put(a[0], [_known(lambda x, y, z: x * y + z, *w) for w in zip(*(self.lanes(t) for t in a[2:5]))])
        elif re.match(r"v_cmp_(eq|ne|lt|le|gt|ge)_[iu]32$", op):
            f = COMPARE[op[6:8]] if op[-3] == "u" else lambda x, y: COMPARE[op[6:8]](_signed(x & M32), _signed(y & M32))
            bits = [_known(f, x, y) for n, (x, y) in enumerate(zip(self.lanes(a[1]), self.lanes(a[2]))) if self.flag["exec"] >> n & 1]
            where = [n for n in range(64) if self.flag["exec"] >> n & 1]
            self.put(a[0], None if None in bits else sum(int(b) << n for n, b in zip(where, bits)))
        else:
            self.forget(op, a)


def _args(code, T, E, k, score, bias, groups, top_groups, best, renorm):
    """The kernel's arguments as 32-bit words by their offset."""
    layout = [(0, LOGITS), (8, T), (12, E), (16, k), (20, score), (24, BIAS if bias else 0), (32, groups), (36, top_groups), (40, best), (44, renorm),
              (48, None), (56, IDS), (64, WEIGHTS)]
    words = {code.group_size: 64}
    for at, v in layout:
        words[at] = None if v is None else v & M32
        if at in (0, 24, 56, 64):
            words[at + 4] = v >> 32
    return words


def _check(code, bias, size, E, t, k, groups, score, renorm, rng):
    where = (bias, size, E, t, k, groups, score, renorm)
    args = _args(code, t + 2, E, k, score, bias, groups, max(1, groups // 2), 2, renorm)
    read, wrote = {LOGITS: [], BIAS: []}, {IDS: [], WEIGHTS: []}
    for store, addresses in Wave(code, args, t, rng).walk():
        assert None not in addresses, (where, "store" if store else "load", "an address that nothing defines")
        for x in addresses:
            (wrote if store else read).setdefault(x >> 36 << 36, []).append(x & (1 << 36) - 1)
    assert sorted(read[LOGITS]) == [(t * E + e) * size for e in range(E)], where
    assert sorted(read[BIAS]) == ([4 * e for e in range(E)] if bias else []), where
    for base in (IDS, WEIGHTS):
        assert sorted(wrote[base]) == [4 * (t * k + j) for j in range(k)], where
    assert len(read) == 2 and len(wrote) == 2, where


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    flags = subprocess.run(["make", "-s", "-C", CSRC, "flags"], capture_output=True, text=True, check=True).stdout.split()
    out = str(tmp_path_factory.mktemp("route") / "route.s")
    cc = subprocess.run([HIPCC, *flags, "--offload-device-only", "-S", os.path.join(CSRC, "route.hip"), "-o", out], capture_output=True, text=True)
    assert cc.returncode == 0, cc.stderr[-3000:]
    with open(out) as f:
        text = f.read()
    found = {}
    for name, per, bias, ldt, body, kd in re.findall(r"^(_ZN\S*route_kernelILi(\d+)ELb(\d)ELi(\d)E\S*):[^\n]*\n(.*?)^\t\.section\t\.rodata(.*?)\.end_amdhsa_kernel", text, re.M | re.S):
        meta = text[:text.index(f".name:           {name}\n")].rpartition("  - .agpr_count")[2]
        found[int(per), int(bias), int(ldt)] = Code(body, kd, meta)
    return found


@pytest.mark.parametrize("per,lo,hi", [(1, 1, 64), (2, 65, 128), (4, 129, 256), (8, 257, 512), (16, 513, 1024)])
@pytest.mark.parametrize("bias", [0, 1])
def test_every_address_is_defined_and_within_its_array(kernels, per, lo, hi, bias):
    assert len(kernels) == 30
    rng = random.Random(per * 2 + bias)
    for ldt, size in ((0, 4), (1, 2), (2, 2)):
        sizes = {lo, hi, rng.randint(lo, hi), rng.randint(lo, hi) // 8 * 8 or 8} | ({1000} if per == 16 else set())
        for E in sorted(e for e in sizes if lo <= e <= hi):
            for groups in (1, 8) if E % 8 == 0 else (1,):
                _check(kernels[per, bias, ldt], bias, size, E, rng.choice((0, 5)), min(E // groups, 3), groups, rng.randint(0, 1), rng.randint(0, 1), rng)

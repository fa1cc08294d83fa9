"""Which bytes the head's tiled products read, from the launches that the library's host code makes.

Run as a program in a process of its own (no torch: its HIP runtime must not be loaded): launch_reach.py RECORDER LIBRARY,
a JSON list of calls on stdin, one JSON list of complaints on stdout.  The addresses are made up: nothing is executed."""
import ctypes
import json
import re
import struct
import sys

import numpy as np

ELEM = {"float": 4, "half": 2, "wino::bf16_t": 2, "wino::mx4_t": 0}
K_INNER, K_OUTER = 0, 1


def operand(raw):
    p, scale, pitch, step, rows, pieces = struct.unpack("<QQqqii", raw)
    return dict(p=p, scale=scale, pitch=pitch, step=step, rows=rows, pieces=pieces)


def tile_args(text):
    raw = bytes.fromhex(text)
    names = ("M", "N", "K", "passes", "a_turn", "b_turn", "mt", "nt", "stages", "split", "pass", "tail_at")
    return dict(zip(names, struct.unpack("<iiiiqqiiiiii", raw[80:136])), a=operand(raw[:40]), b=operand(raw[40:80]))


def kernels(name):
    """(type, order of A, order of B, BM, BN, RB) of the products in a launch, in the order of their arguments."""
    m = re.search(r"tile_gemm_kernel<([^,]+), (\d+), (\d+), (\d+), (\d+), (\d+), (\d+), (\d+),", name)
    if m:
        return [(m[1],) + tuple(int(m[i]) for i in (2, 3, 4, 5, 8))]
    m = re.search(r"ce_gradients_kernel<([^>,]+)>", name)
    return [(m[1], K_OUTER, K_INNER, 64, 64, 128), (m[1], K_OUTER, K_OUTER, 64, 64, 128)] if m else []


def offsets(op, order, elem, ext, rb, org, k_left):
    """Bytes from the stage's base at which a workgroup's 16-byte loads of one operand start: the kernel's arithmetic."""
    at = np.arange(0, ext * rb, 16, dtype=np.int64)
    pieces = rb // 16
    if order == K_INNER:
        row = at // rb
        c = np.minimum(((at // 16) % pieces) ^ ((row // (16 // pieces)) & (pieces - 1)), k_left - 1)
        return np.maximum(np.minimum(row, op["rows"] - 1 - org), 0) * op["pitch"] + c * 16
    k_row, steps = ext * elem, pieces // 2
    krow, c = at // k_row, (at % k_row) >> 4
    inside = k_row // 16 - 1
    c = c ^ (((krow // (4 * steps)) & 1) * 8 & inside) if elem == 4 else c ^ (((krow & 3) * 4) & inside)
    return np.minimum(krow, k_left - 1) * op["pitch"] + np.minimum(c, op["pieces"] - 1 - org // (16 // elem)) * 16


def operand_reach(g, op, turn, order, elem, ext, rb, tiles, two):
    """(lowest, highest + 1) address of the operand that the launch reads, over all tiles and stages."""
    piece = 16 // elem if elem else 32
    stage = rb // 16 * piece
    lo, hi = 1 << 62, 0
    for t in sorted({0, tiles // 2, tiles - 1}):
        org = t * ext
        origin = org * elem if order == K_OUTER else min(org, op["rows"] - 1) * op["pitch"]
        for s in sorted({0, g["pass"] - 1, min(g["pass"], g["stages"] - 1), g["stages"] - 1}):
            second = two and s >= g["pass"]
            local = s - g["pass"] if second else s
            base = op["p"] + origin + s * op["step"] + (turn if second else 0)
            left = 1 << 30 if order == K_OUTER else rb // 16
            if local == g["tail_at"]:
                k0 = local * stage
                left = op["rows"] - k0 if order == K_OUTER else min(left, -(-(g["K"] - k0) // piece))
            off = offsets(op, order, elem, ext, rb, org, left)
            assert off.min() >= 0 and off.max() < 1 << 32
            lo, hi = min(lo, base + int(off.min())), max(hi, base + int(off.max()) + 16)
    return lo, hi


def complaints(call, records, buffers):
    found = []
    for line in records.strip().split("\n"):
        name, grid, args = line.split("|")
        gx, gy, gz, block = map(int, grid.split())
        if gx * block >= 1 << 32:
            found.append(f"{call}: {name[:80]}: {gx} x {block} threads")
        products = kernels(name)
        assert len(products) == len(args.split()), f"not understood: {name}"
        for (kind, ao, bo, bm, bn, rb), text in zip(products, args.split()):
            g, elem = tile_args(text), ELEM[kind]
            two = ao == K_OUTER and elem == 2
            assert two or g["passes"] == 1
            for which, order, ext, tiles, turn in (("a", ao, bm, g["mt"], g["a_turn"]), ("b", bo, bn, g["nt"], g["b_turn"])):
                op = g[which]
                lo, hi = operand_reach(g, op, turn, order, elem, ext, rb, tiles, two)
                size = g["stages"] * op["step"] if kind == "wino::mx4_t" else op["rows"] * op["pitch"]
                end = op["p"] + size
                if lo < op["p"] or hi > end:
                    found.append(f"{call}: {name[:60]} operand {which} reads [{lo - op['p']}, {hi - op['p']}) of {size} bytes")
                if not any(b <= op["p"] and end <= e for b, e in buffers):
                    found.append(f"{call}: {name[:60]} operand {which} lies outside the call's buffers")
    return found


def run(lib, recorder, call):
    X, W, B, Y, WS, OTHER = (1 + np.arange(6, dtype=object)) << 44
    kind, dt, a, b, c = call
    recorder.forget()
    V, S = ctypes.c_void_p, ctypes.c_size_t
    e = 4 if dt == 0 else 2
    if kind == "linear":
        M, N, K = a, b, c
        kp = (K + 127) // 128 * 128
        lib.wino_mx4_workspace_bytes.restype = S
        n = lib.wino_mx4_workspace_bytes(M, N, K)
        rc = lib.wino_mx4_linear(dt, 0, M, N, K, V(X), V(W), V(OTHER), None, V(Y), V(WS), S(n), None)
        buffers = [(X, X + M * K * e), (W, W + N * kp // 2), (WS, WS + n)]
    else:
        T, D, Vo = a, b, c
        lib.wino_linear_cross_entropy_workspace_bytes.restype = S
        back = int(kind == "backward")
        n = lib.wino_linear_cross_entropy_workspace_bytes(dt, T, D, Vo, V(X), V(W), back)
        head = (dt, T, D, Vo, V(X), V(W), V(B), V(OTHER), ctypes.c_longlong(-100))
        if back:
            rc = lib.wino_linear_cross_entropy_backward(*head, V(OTHER), V(OTHER), V(Y), V(Y), V(Y), V(WS), S(n), None)
        else:
            rc = lib.wino_linear_cross_entropy(*head, V(OTHER), V(OTHER), V(WS), S(n), None)
        buffers = [(X, X + T * D * e), (W, W + Vo * D * e), (WS, WS + n)]
    if rc:
        lib.wino_last_error.restype = ctypes.c_char_p
        return [f"{call}: {lib.wino_last_error().decode()}"]
    recorder.recorded.restype = ctypes.c_char_p
    return complaints(call, recorder.recorded().decode(), buffers)


if __name__ == "__main__":
    rec = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
    wino = ctypes.CDLL(sys.argv[2])
    print(json.dumps([c for call in json.load(sys.stdin) for c in run(wino, rec, tuple(call))]))

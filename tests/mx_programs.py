"""Random programs of microscaled and plain steps over a small pool of slots: later steps overwrite
what earlier ones read or wrote, and products of at least 2^28 multiply-adds make the two-stream
schedule active. Every slot is written before it is read."""
import numpy as np

from synaptik_amd.program import ProgramBuilder

N = 64
BIG = 700
FORMATS = ["e4m3", "e5m2", "e2m1"]


def random_program(seed):
    """(builder, input arrays in order, output slots)."""
    rng = np.random.default_rng(seed)
    pb = ProgramBuilder()
    arrays = [rng.standard_normal(N * N).astype(np.float32), rng.standard_normal(BIG * BIG).astype(np.float32)]
    small_in, big_in = pb.input(N * N), pb.input(BIG * BIG)
    small_out, big_out, sums = pb.output(N * N), pb.output(BIG * BIG), pb.output(N)
    sizes = {"small": N, "big": BIG}
    wide = {"small": [small_out] + [pb.internal(N * N) for _ in range(3)],
            "big": [big_out, pb.internal(BIG * BIG)]}
    kept = {k: [(f, pb.mx_tensor(n, n, f)) for f in FORMATS] for k, n in sizes.items()}
    ready = {"small": [small_in], "big": [big_in]}

    def pick(pool):
        return pool[int(rng.integers(len(pool)))]

    def wrote(k, slot):
        if slot not in ready[k]:
            ready[k].append(slot)

    # everything has a value: encoded inputs, copies of them, sums
    for k, n in sizes.items():
        for f, t in kept[k]:
            pb.mx_encode(ready[k][0], t, n, n, format=f)
        for slot in wide[k]:
            pb.copy(ready[k][0], slot, n * n)
            wrote(k, slot)
    pb.colsum(small_in, sums, N, N)
    for _ in range(int(rng.integers(10, 24))):
        k = "big" if rng.random() < 0.3 else "small"
        n = sizes[k]
        src, dst, (f, t) = pick(ready[k]), pick(wide[k]), pick(kept[k])
        op = int(rng.integers(0, 9))
        if op == 0:
            pb.mx_encode(src, t, n, n, format=f)
        elif op == 1:
            pb.mx_decode(t, dst, n, n, format=f)
        elif op == 2:  # in place as well
            pb.mx_act_grad(src, t, dst, n, n, act="relu", format=f, colsum=sums if k == "small" else None)
        elif src is dst:
            continue
        elif op in (3, 4):
            pb.mx_gemm(src, t, dst, n, n, n, format=f, trans_a=bool(rng.integers(2)))
        elif op in (5, 6):
            pb.mx_linear(src, t, dst, n, n, n, w_format=f, x_format=pick(FORMATS),
                         bias=sums if k == "small" else None, act=pick([None, "tanh"]))
        elif op == 7:
            pb.gemm(src, pick([s for s in ready[k] if s is not dst]), dst, n, n, n, trans_b=True, act="tanh")
        else:
            pb.colsum(small_in, sums, N, N)
    return pb, arrays, [small_out, big_out, sums]

"""What rotary positions, tables of pages and attention to chosen pages would launch, seen on the CPU: run as a program with the launch recorder
preloaded, it reads a list of calls as JSON and prints, for each, its status and its launches.  launches() builds the recorder and runs it."""
import ctypes
import json
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
A = 0x100000  # an address that nothing reaches: no launch is made


def launches(tmp_path, calls):
    """calls: (kind, sizes ...), as the functions below take them.  Returns a list of dicts: status, launches."""
    so = str(tmp_path / "librecorder.so")
    if not os.path.exists(so):
        subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(HERE, "cpp", "launch_recorder.cpp"), "-o", so])
    env = dict(os.environ, LD_PRELOAD=so, RECORDER=so, CUDA_VISIBLE_DEVICES="", HIP_VISIBLE_DEVICES="")
    out = subprocess.run([sys.executable, os.path.abspath(__file__)], input=json.dumps(calls), capture_output=True, text=True, env=env, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    return json.loads(out.stdout.splitlines()[-1])


def main():
    sys.path.insert(0, HERE)
    from attention_reference import load_abq_attention
    attn = load_abq_attention()
    L, rec = attn.lib(), ctypes.CDLL(os.environ["RECORDER"])
    rec.recorder_name.restype = ctypes.c_char_p
    ref = ctypes.byref

    def recorded():
        made = []
        for i in range(rec.recorder_count()):
            grid, block, lds = (ctypes.c_uint32 * 3)(), (ctypes.c_uint32 * 3)(), ctypes.c_uint64()
            rec.recorder_sizes(i, grid, block, ref(lds))
            made.append({"kernel": rec.recorder_name(i).decode(), "grid": list(grid), "block": list(block), "lds": lds.value})
        return made

    def cache(kv, dim=128, size=16, pages=1000):
        return attn.KvCacheDesc(8, 1, kv, dim, size, pages, A, A, A, A)

    def rows(n, heads, dim, at=A):
        return attn.Rows(at, n, heads * dim, dim)

    def rotary(n, heads, kv, dim):
        q, k = rows(n, heads, dim), rows(n, max(kv, 1), dim, 2 * A)
        return L.abq_rotary_apply(ref(attn.RotaryDesc(dim, 1, 0, A, None)), ref(q), ref(q), heads, ref(k) if kv else None, ref(k) if kv else None, kv, dim, 0, A, n, None)

    def append(n, heads, kv, dim):
        q, k, v = rows(n, heads, dim), rows(n, kv, dim, 2 * A), rows(n, kv, dim, 3 * A)
        return L.abq_kv_append_rotary(ref(cache(kv, dim)), ref(attn.RotaryDesc(dim, 1, 0, A, None)), ref(q), ref(q), heads, ref(k), None, ref(v), 0, A, n, A, None)

    def pages(seqs, most, num=1 << 20):
        return ref(attn.KvPagesDesc(seqs, most, 16, num, A, A, A))

    def choose(kv, seqs, max_q, columns, max_context):
        c, q = cache(kv), rows(seqs * max_q, 4 * kv, 128)
        need = L.abq_attn_choose_workspace_bytes(ref(c), columns, seqs, max_q, max_context)
        return L.abq_attn_choose(ref(c), ref(attn.KvBoundsDesc(A, A)), ref(q), 0, 4 * kv, A, columns, A, A, seqs, max_q, max_context, 1, 1, 50, A, A if need else None, need, None)

    def sparse(kv, seqs, max_q, columns, max_context):
        st, q = attn.SparseState(), rows(seqs * max_q, 4 * kv, 128)
        rc = L.abq_attn_sparse_init(ref(cache(kv)), ref(q), ref(q), 0, 4 * kv, A, columns, A, A, None, A, columns // 2, seqs, max_q, max_context, 0.1, ref(st))
        if rc == 0:
            rc = L.abq_attn_sparse_set_workspace(ref(st), A, L.abq_attn_sparse_workspace_bytes(ref(st)))
        return rc or L.abq_attn_sparse_exec(ref(st), None)

    kinds = {"rotary": rotary, "append": append, "choose": choose, "sparse": sparse,
             "fork": lambda seqs, most: L.abq_kv_pages_fork(pages(seqs, most), A, None),
             "extend": lambda seqs, most, n: L.abq_kv_pages_extend(pages(seqs, most), A, A, n, A, A, A, None),
             "compact": lambda seqs, most: L.abq_kv_pages_compact(pages(seqs, most), A, None),
             "copy": lambda kv, n: L.abq_kv_copy_pages(ref(cache(kv)), None, A, n, None),
             "bound": lambda kv, n: L.abq_kv_bound(ref(cache(kv)), ref(attn.KvBoundsDesc(A, A)), A, n, None)}

    def one(call):
        rec.recorder_clear()
        return {"status": kinds[call[0]](*call[1:]), "launches": recorded()}

    print(json.dumps([one(c) for c in json.load(sys.stdin)]))


if __name__ == "__main__":
    main()

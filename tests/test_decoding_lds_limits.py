"""What launches around the quantised cache ask for of LDS, seen on the CPU.  The limit that a kernel is allowed belongs to the process: a call
that lowered it could do so between another thread's raising it and its launch."""
import ctypes
import json
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
A = 0x100000  # an address that nothing reaches: no launch is made
UNASKED = 64 << 10  # bytes that every launch gets


def test_no_call_lowers_what_another_launches_with(tmp_path):
    so = str(tmp_path / "liblimits.so")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(HERE, "cpp", "lds_limit_recorder.cpp"), "-o", so])
    env = dict(os.environ, LD_PRELOAD=so, RECORDER=so, CUDA_VISIBLE_DEVICES="", HIP_VISIBLE_DEVICES="")
    out = subprocess.run([sys.executable, os.path.abspath(__file__)], capture_output=True, text=True, env=env, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    limits, seen = {}, 0
    for call in json.loads(out.stdout.splitlines()[-1]):
        assert call["status"] == 0, call
        for name, value in call["limits"]:
            assert value >= limits.get(name, 0), (name, value, limits[name])
            limits[name] = value
        for name, lds in call["launches"]:
            assert lds <= limits.get(name, UNASKED), (name, lds)
            seen = max(seen, lds)
    assert seen == 128 << 10 and limits


def main():
    sys.path.insert(0, HERE)
    from attention_reference import load_abq_attention
    attn = load_abq_attention()
    L, rec, ref = attn.lib(), ctypes.CDLL(os.environ["RECORDER"]), ctypes.byref
    rec.recorder_name.restype = rec.limit_name.restype = ctypes.c_char_p

    def choose(columns, seqs, max_context, dim):
        c, q = attn.KvCacheDesc(8, 1, 8, dim, 16, 1000, A, A, A, A), attn.Rows(A, seqs, 32 * dim, dim)
        need = L.abq_attn_choose_workspace_bytes(ref(c), columns, seqs, 1, max_context)
        return L.abq_attn_choose(ref(c), ref(attn.KvBoundsDesc(A, A)), ref(q), 0, 32, A, columns, A, A, seqs, 1, max_context, 1, 1, 50, A, A if need else None, need, None)

    def fork(seqs):
        return L.abq_kv_pages_fork(ref(attn.KvPagesDesc(seqs, 9, 16, 1000, A, A, A)), A, None)

    said = []
    calls = [lambda n=n, s=s, c=c, d=d: choose(n, s, c, d) for d in (64, 128) for s, c in ((1, 1 << 19), (8, 1 << 19), (40, 9000), (80, 4000), (900, 0))
             for n in (32768, 12300, 16000, 20000, 12288, 32768, 13000)]
    for call in calls + [lambda s=s: fork(s) for s in (1, 4096, 4097, 8192, 3)]:
        rec.recorder_clear()
        before, status = rec.limit_count(), call()
        launches = []
        for i in range(rec.recorder_count()):
            lds = ctypes.c_uint64()
            rec.recorder_sizes(i, (ctypes.c_uint32 * 3)(), (ctypes.c_uint32 * 3)(), ref(lds))
            launches.append((rec.recorder_name(i).decode(), lds.value))
        said.append({"status": status, "launches": launches, "limits": [(rec.limit_name(i).decode(), rec.limit_value(i)) for i in range(before, rec.limit_count())]})
    print(json.dumps(said))


if __name__ == "__main__":
    main()

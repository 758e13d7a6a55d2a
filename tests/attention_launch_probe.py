"""What a call of attention would launch, seen on the CPU: run as a program with the launch recorder preloaded, it reads a list of
calls as JSON and prints, for each, its statuses, its state and its launches.  launches() builds the recorder and runs it."""
import ctypes
import json
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
A = 0x100000  # an address that nothing reaches: no launch is made


def launches(tmp_path, calls):
    """calls: dicts of kind ("tree" or "prompt"), rows, heads, kv_heads, dim, seqs, max_q, max_k (tree: of the context) and optionally
    workspace (bytes; by default what the state asks for).  Returns a list of dicts: status, parts, block_rows, need, launches."""
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

    def recorded():
        made = []
        for i in range(rec.recorder_count()):
            grid, block, lds = (ctypes.c_uint32 * 3)(), (ctypes.c_uint32 * 3)(), ctypes.c_uint64()
            rec.recorder_sizes(i, grid, block, ctypes.byref(lds))
            made.append({"kernel": rec.recorder_name(i).decode(), "grid": list(grid), "block": list(block)})
        return made

    def one(c):
        rec.recorder_clear()
        st, dim, kv = attn.AttnState(), c.get("dim", 128), c["kv_heads"]
        q, k = attn.Rows(A, c["rows"], c["heads"] * dim, dim), attn.Rows(A, c["rows"], kv * dim, dim)
        r = [ctypes.byref(x) for x in (q, k)]
        if c["kind"] == "tree":
            cache = attn.KvCacheDesc(8, 1, kv, dim, 64, 1000, A, A, A, A)
            rc = [L.abq_attn_tree_init(ctypes.byref(cache), r[0], r[0], 0, c["heads"], A, 1000, A, A, None, c["seqs"], c["max_q"], c["max_k"], 0.1,
                                       ctypes.byref(st))]
        else:
            rc = [L.abq_attn_prompt_init(r[0], r[1], r[1], r[0], 0, c["heads"], kv, dim, A, A, c["seqs"], c["max_q"], c["max_k"], 0.1, ctypes.byref(st))]
        need = L.abq_attn_workspace_bytes(ctypes.byref(st))
        rc.append(L.abq_attn_set_workspace(ctypes.byref(st), A, c.get("workspace", need)))
        rc.append(L.abq_attn_exec(ctypes.byref(st), None))
        return {"status": rc, "parts": st.parts, "block_rows": st.block_rows, "need": need, "launches": recorded()}

    print(json.dumps([one(c) for c in json.load(sys.stdin)]))


if __name__ == "__main__":
    main()

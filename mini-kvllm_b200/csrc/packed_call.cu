// The tree and cache-copy calls with their arguments as an array of 64-bit words (mkv_call_packed in
// include/mkv.h): 12 to 22 us of a call from Python became 6 to 8 (ctypes converts each argument).
#include <cstring>

#include "mkv_common.cuh"

using namespace mkv;

namespace {
struct Args {
  const int64_t* a;
  int i = 0;
  template <typename T> T* ptr() { return reinterpret_cast<T*>(a[i++]); }
  int32_t i32() { return (int32_t)a[i++]; }
  int64_t i64() { return a[i++]; }
  float f32() {
    double d;
    memcpy(&d, a + i++, 8);
    return (float)d;
  }
};
}  // namespace

// Each call reads its words into named values first: the order in which function arguments are
// evaluated is not fixed.
extern "C" int mkv_call_packed(int32_t call, const int64_t* args) {
  clear_error();
  if (!args) return set_error(MKV_ERR_INVALID_ARGUMENT, "mkv_call_packed: null pointer argument");
  Args x{args};
  switch (call) {
    case MKV_CALL_PAGED_TREE_ATTENTION:
    case MKV_CALL_PAGED_TREE_ATTENTION + MKV_CALL_ZEROED: {
      const void* q = x.ptr<const void>();
      const int64_t qst = x.i64(), qsh = x.i64();
      const int32_t qdt = x.i32();
      const void* k = x.ptr<const void>();
      const void* v = x.ptr<const void>();
      const int32_t cdt = x.i32();
      const float* ks = x.ptr<const float>();
      const float* vs = x.ptr<const float>();
      const float* kss = x.ptr<const float>();
      const float* vss = x.ptr<const float>();
      const int64_t nb = x.i64();
      const int32_t bs = x.i32();
      const void* bt = x.ptr<const void>();
      const int32_t btt = x.i32();
      const int64_t bts = x.i64();
      const int32_t maxb = x.i32();
      const void* cl = x.ptr<const void>();
      const int32_t clt = x.i32();
      const void* cu = x.ptr<const void>();
      const int32_t cut = x.i32();
      const uint64_t* mask = x.ptr<const uint64_t>();
      const int64_t mst = x.i64();
      const int32_t words = x.i32(), B = x.i32();
      const int64_t T = x.i64();
      const int32_t H = x.i32(), KVH = x.i32(), D = x.i32();
      const float scale = x.f32();
      void* out = x.ptr<void>();
      const int64_t ost = x.i64(), osh = x.i64();
      void* ws = x.ptr<void>();
      const size_t wsb = (size_t)x.i64();
      void* stream = x.ptr<void>();
      const auto fn = call & MKV_CALL_ZEROED ? mkv_paged_tree_attention_zeroed : mkv_paged_tree_attention;
      return fn(q, qst, qsh, qdt, k, v, cdt, ks, vs, kss, vss, nb, bs, bt, btt, bts, maxb, cl, clt, cu, cut, mask, mst,
                words, B, T, H, KVH, D, scale, out, ost, osh, ws, wsb, stream);
    }
    case MKV_CALL_TREE_METADATA:
    case MKV_CALL_TREE_ACCEPT: {
      const bool accept = call == MKV_CALL_TREE_ACCEPT;
      const void* draft = accept ? x.ptr<const void>() : nullptr;
      const void* target = accept ? x.ptr<const void>() : nullptr;
      const int32_t tokt = accept ? x.i32() : 0;
      const void* par = x.ptr<const void>();
      const int32_t pt = x.i32();
      const void* cu = x.ptr<const void>();
      const int32_t cut = x.i32();
      const void* pre = x.ptr<const void>();
      const int32_t pret = x.i32();
      const void* bt = x.ptr<const void>();
      const int32_t btt = x.i32();
      const int64_t bts = x.i64();
      const int32_t maxb = x.i32(), bs = x.i32(), B = x.i32();
      const int64_t T = x.i64();
      const int32_t n = x.i32();  // mask_words or max_path
      if (!accept) {
        int64_t* slots = x.ptr<int64_t>();
        int64_t* lens = x.ptr<int64_t>();
        int64_t* pos = x.ptr<int64_t>();
        uint64_t* mask = x.ptr<uint64_t>();
        int32_t* bad = x.ptr<int32_t>();
        void* stream = x.ptr<void>();
        return mkv_tree_metadata(par, pt, cu, cut, pre, pret, bt, btt, bts, maxb, bs, B, T, n, slots, lens, pos, mask, bad,
                                 stream);
      }
      int32_t* count = x.ptr<int32_t>();
      int32_t* nodes = x.ptr<int32_t>();
      int64_t* tokens = x.ptr<int64_t>();
      int64_t* lens = x.ptr<int64_t>();
      int64_t* src = x.ptr<int64_t>();
      int64_t* dst = x.ptr<int64_t>();
      void* stream = x.ptr<void>();
      return mkv_tree_accept(draft, target, tokt, par, pt, cu, cut, pre, pret, bt, btt, bts, maxb, bs, B, T, n, count,
                             nodes, tokens, lens, src, dst, stream);
    }
    case MKV_CALL_COPY_KV_PAGES:
    case MKV_CALL_MOVE_KV_ROWS: {
      void* k = x.ptr<void>();
      void* v = x.ptr<void>();
      const int32_t cdt = x.i32(), L = x.i32();
      const int64_t ls = x.i64(), nb = x.i64();
      const int32_t bs = x.i32(), KVH = x.i32(), D = x.i32();
      float* ks = x.ptr<float>();
      float* vs = x.ptr<float>();
      const int64_t ss = x.i64();
      const void* src = x.ptr<const void>();
      const void* dst = x.ptr<const void>();
      const int32_t it = x.i32();
      if (call == MKV_CALL_COPY_KV_PAGES) {
        const int64_t n = x.i64();
        int32_t* bad = x.ptr<int32_t>();
        void* stream = x.ptr<void>();
        return mkv_copy_kv_pages(k, v, cdt, L, ls, nb, bs, KVH, D, ks, vs, ss, src, dst, it, n, bad, stream);
      }
      const int32_t G = x.i32(), M = x.i32();
      int32_t* bad = x.ptr<int32_t>();
      void* stream = x.ptr<void>();
      return mkv_move_kv_rows(k, v, cdt, L, ls, nb, bs, KVH, D, ks, vs, ss, src, dst, it, G, M, bad, stream);
    }
    default:
      return set_error(MKV_ERR_INVALID_ARGUMENT, "mkv_call_packed: unknown call %d", call);
  }
}

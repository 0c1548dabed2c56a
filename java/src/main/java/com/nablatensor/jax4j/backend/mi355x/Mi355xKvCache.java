package com.nablatensor.jax4j.backend.mi355x;

import static java.lang.foreign.ValueLayout.JAVA_BYTE;
import static java.lang.foreign.ValueLayout.JAVA_FLOAT;
import static java.lang.foreign.ValueLayout.JAVA_INT;
import static java.lang.foreign.ValueLayout.JAVA_LONG;

import java.lang.foreign.Arena;
import java.lang.foreign.MemorySegment;
import java.lang.ref.Cleaner;
import java.util.Queue;
import java.util.concurrent.ConcurrentLinkedQueue;
import java.util.concurrent.atomic.AtomicBoolean;

/**
 * A paged 8-bit key/value cache and the attention that reads it (j4q_kv_*), for what a decoder does between its q|k|v and
 * o projections. Engine-local: the reference has no attention. Arguments that are addresses (of queries, keys, values,
 * results, rotary tables) are device addresses as {@link Mi355xBackend#devicePointer} gives them, and the caller keeps
 * what they belong to reachable until a sync; calls enqueue on the engine stream and do not wait.
 *
 * <p>A step: {@link #extend} names the sequences and how many tokens each gets, then per layer {@link #append} and
 * {@link #attend} over these tokens, in that order.
 *
 * <p>{@link #close()} waits for the device and frees the cache; an unreachable cache is freed on the backend's next call.
 */
public final class Mi355xKvCache implements AutoCloseable {
  private static final Cleaner CLEANER = Cleaner.create();
  private static final Queue<Long> PENDING = new ConcurrentLinkedQueue<>();

  private static final class State implements Runnable {
    final long handle;
    final AtomicBoolean closed = new AtomicBoolean();

    State(long handle) {
      this.handle = handle;
    }

    @Override
    public void run() {
      if (closed.compareAndSet(false, true)) PENDING.add(handle);
    }
  }

  /**
   * Rotary positions: tables of cosines and sines [rows, dims / 2] (device, fp32), positions [axes, rows] (device, int32;
   * 0: a token's place in its sequence) and the axis of each pair (null: one axis).
   */
  public record Rope(long cos, long sin, long rows, int dims, boolean interleaved, long positions, byte[] pairAxis) {
    MemorySegment segment(Arena a) {
      if (pairAxis != null && 2 * pairAxis.length != dims)
        throw new IllegalArgumentException(pairAxis.length + " pairs with axes, for " + dims + " rotary channels");
      MemorySegment s = a.allocate(48, 8);
      s.set(JAVA_LONG, 0, cos);
      s.set(JAVA_LONG, 8, sin);
      s.set(JAVA_LONG, 16, rows);
      s.set(JAVA_INT, 24, dims);
      s.set(JAVA_INT, 28, interleaved ? 1 : 0);
      s.set(JAVA_LONG, 32, positions);
      s.set(JAVA_LONG, 40, pairAxis == null ? 0 : a.allocateFrom(JAVA_BYTE, pairAxis).address());
      return s;
    }
  }

  private final int sequencePages;
  private final State state;
  private final Cleaner.Cleanable cleanable;

  Mi355xKvCache(long handle, int sequencePages) {
    this.sequencePages = sequencePages;
    this.state = new State(handle);
    this.cleanable = CLEANER.register(this, state);
  }

  /** j4q_kv_config. */
  static MemorySegment config(Arena a, int layers, int kvHeads, int headDim, int pageTokens, long pages, int sequences, int sequencePages) {
    MemorySegment s = a.allocate(32, 8);
    s.set(JAVA_INT, 0, layers);
    s.set(JAVA_INT, 4, kvHeads);
    s.set(JAVA_INT, 8, headDim);
    s.set(JAVA_INT, 12, pageTokens);
    s.set(JAVA_LONG, 16, pages);
    s.set(JAVA_INT, 24, sequences);
    s.set(JAVA_INT, 28, sequencePages);
    return s;
  }

  private long handle() {
    if (state.closed.get()) throw new IllegalStateException("key/value cache is closed");
    return state.handle;
  }

  private static void equal(int a, int b, String what) {
    if (a != b) throw new IllegalArgumentException(a + " sequences, " + b + " " + what);
  }

  // ---- pages -------------------------------------------------------------------------------

  /** Begins a step: sequence seqs[i] gets tokens[i] more tokens (the step's rows, in this order). */
  public void extend(int[] seqs, int[] tokens) {
    equal(seqs.length, tokens.length, "counts of tokens");
    try (Arena a = Arena.ofConfined()) {
      Mi355xNative.call("kvExtend", Mi355xNative.KV_EXTEND, handle(), a.allocateFrom(JAVA_INT, seqs), a.allocateFrom(JAVA_INT, tokens),
          seqs.length, MemorySegment.NULL);
    }
  }

  /** Begins a step over the last tokens[i] tokens that sequence seqs[i] has already. */
  public void begin(int[] seqs, int[] tokens) {
    equal(seqs.length, tokens.length, "counts of tokens");
    try (Arena a = Arena.ofConfined()) {
      Mi355xNative.call("kvBegin", Mi355xNative.KV_BEGIN, handle(), a.allocateFrom(JAVA_INT, seqs), a.allocateFrom(JAVA_INT, tokens),
          seqs.length, MemorySegment.NULL);
    }
  }

  /** The empty sequence dst[i] becomes src[i], sharing its pages or with copies of them. */
  public void fork(int[] src, int[] dst, boolean share) {
    equal(src.length, dst.length, "forks");
    try (Arena a = Arena.ofConfined()) {
      Mi355xNative.call("kvFork", Mi355xNative.KV_FORK, handle(), a.allocateFrom(JAVA_INT, src), a.allocateFrom(JAVA_INT, dst), src.length,
          share ? 1 : 0, MemorySegment.NULL);
    }
  }

  /** Cuts sequences to lengths[i] tokens; 0 frees them. */
  public void truncate(int[] seqs, long[] lengths) {
    equal(seqs.length, lengths.length, "lengths");
    try (Arena a = Arena.ofConfined()) {
      Mi355xNative.call("kvTruncate", Mi355xNative.KV_TRUNCATE, handle(), a.allocateFrom(JAVA_INT, seqs), a.allocateFrom(JAVA_LONG, lengths),
          seqs.length);
    }
  }

  /** Frees the pages that no later token sees through a window of so many tokens and so many first ones. */
  public void evict(int[] seqs, int window, int sinks) {
    try (Arena a = Arena.ofConfined()) {
      Mi355xNative.call("kvEvict", Mi355xNative.KV_EVICT, handle(), a.allocateFrom(JAVA_INT, seqs), seqs.length, window, sinks,
          MemorySegment.NULL);
    }
  }

  /** Moves pages so that those in use are the pool's lowest; how many were moved. */
  public long compact() {
    try (Arena a = Arena.ofConfined()) {
      MemorySegment moved = a.allocate(JAVA_LONG);
      Mi355xNative.call("kvCompact", Mi355xNative.KV_COMPACT, handle(), moved, MemorySegment.NULL);
      return moved.get(JAVA_LONG, 0);
    }
  }

  /** Tokens of the sequences. */
  public long[] lengths(int[] seqs) {
    try (Arena a = Arena.ofConfined()) {
      MemorySegment out = a.allocate(JAVA_LONG, seqs.length);
      Mi355xNative.call("kvTables", Mi355xNative.KV_TABLES, handle(), a.allocateFrom(JAVA_INT, seqs), seqs.length, out, MemorySegment.NULL, 0);
      return out.toArray(JAVA_LONG);
    }
  }

  /** Pages of a sequence; -1: evicted, and behind its last page. */
  public int[] pages(int seq) {
    try (Arena a = Arena.ofConfined()) {
      MemorySegment out = a.allocate(JAVA_INT, sequencePages);
      Mi355xNative.call("kvTables", Mi355xNative.KV_TABLES, handle(), a.allocateFrom(JAVA_INT, seq), 1, MemorySegment.NULL, out, sequencePages);
      return out.toArray(JAVA_INT);
    }
  }

  /** Free pages of the pool. */
  public long pagesFree() {
    try (Arena a = Arena.ofConfined()) {
      MemorySegment d = a.allocate(64, 8);
      Mi355xNative.call("kvInfo", Mi355xNative.KV_INFO, handle(), d);
      return d.get(JAVA_LONG, 32);
    }
  }

  // ---- a layer of a step -------------------------------------------------------------------

  /**
   * Stores the step's keys and values, F32 [rows, kv heads, head dim] with `stride` values from a row to the next (0: dense),
   * keys turned by rope (may be null); q (0: none), [rows, heads, head dim], is turned too, in place.
   */
  public void append(int layer, long k, long v, long stride, Rope rope, long q, int heads, long qStride) {
    try (Arena a = Arena.ofConfined()) {
      MemorySegment s = a.allocate(64, 8);
      s.set(JAVA_LONG, 0, k);
      s.set(JAVA_LONG, 8, v);
      s.set(JAVA_LONG, 16, stride);
      s.set(JAVA_INT, 24, Mi355xNative.KIND_F32);
      s.set(JAVA_INT, 28, heads);
      s.set(JAVA_LONG, 32, q);
      s.set(JAVA_LONG, 40, q);
      s.set(JAVA_LONG, 48, qStride);
      s.set(JAVA_LONG, 56, rope == null ? 0 : rope.segment(a).address());
      Mi355xNative.call("kvAppend", Mi355xNative.KV_APPEND, handle(), layer, s, MemorySegment.NULL);
    }
  }

  /**
   * Attention of the step's queries q [rows, heads, head dim] into out, both F32, to the tokens j <= p of their sequence, p their
   * own place, with j > p - window (0: no window) or j < sinks. scale 0: 1 / sqrt(head dim).
   */
  public void attend(int layer, long q, long qStride, long out, long outStride, int heads, int window, int sinks, float scale) {
    attend(layer, q, qStride, Mi355xNative.KIND_F32, out, outStride, Mi355xNative.KIND_F32, heads, window, sinks, scale);
  }

  /** The same into bf16, as the prefill products take it; steps of many tokens are 1.3 to 1.6 times as fast. */
  public void attendBf16(int layer, long q, long qStride, long out, long outStride, int heads, int window, int sinks, float scale) {
    attend(layer, q, qStride, Mi355xNative.KIND_F32, out, outStride, Mi355xNative.KIND_BF16, heads, window, sinks, scale);
  }

  private void attend(int layer, long q, long qStride, int qType, long out, long outStride, int outType, int heads, int window, int sinks,
      float scale) {
    try (Arena a = Arena.ofConfined()) {
      MemorySegment s = a.allocate(56, 8);
      s.set(JAVA_LONG, 0, q);
      s.set(JAVA_LONG, 8, out);
      s.set(JAVA_LONG, 16, qStride);
      s.set(JAVA_LONG, 24, outStride);
      s.set(JAVA_INT, 32, qType);
      s.set(JAVA_INT, 36, outType);
      s.set(JAVA_INT, 40, heads);
      s.set(JAVA_INT, 44, window);
      s.set(JAVA_INT, 48, sinks);
      s.set(JAVA_FLOAT, 52, scale);
      Mi355xNative.call("kvAttend", Mi355xNative.KV_ATTEND, handle(), layer, s, MemorySegment.NULL);
    }
  }

  /** Tokens [first[i], first[i] + count) of seqs[i] as F32 [n, count, kv heads, head dim] at k and v (0: not asked for). */
  public void read(int layer, int[] seqs, long[] first, long count, long k, long v) {
    equal(seqs.length, first.length, "first tokens");
    try (Arena a = Arena.ofConfined()) {
      Mi355xNative.call("kvRead", Mi355xNative.KV_READ, handle(), layer, a.allocateFrom(JAVA_INT, seqs), a.allocateFrom(JAVA_LONG, first), count,
          seqs.length, MemorySegment.ofAddress(k), MemorySegment.ofAddress(v), MemorySegment.NULL);
    }
  }

  /** Waits for the device, then frees the cache; idempotent. */
  @Override
  public void close() {
    if (!state.closed.compareAndSet(false, true)) return;
    Mi355xNative.call("kvDestroy", Mi355xNative.KV_DESTROY, state.handle);
    cleanable.clean();
  }

  static void drainPending() {
    for (Long h; (h = PENDING.poll()) != null; ) {
      try {
        Mi355xNative.status("kvDestroy", Mi355xNative.KV_DESTROY, h.longValue());
      } catch (RuntimeException ignored) {
        // the library is gone: nothing to free
      }
    }
  }
}

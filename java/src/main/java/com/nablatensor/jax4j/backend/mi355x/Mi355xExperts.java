package com.nablatensor.jax4j.backend.mi355x;

import static java.lang.foreign.ValueLayout.JAVA_FLOAT;
import static java.lang.foreign.ValueLayout.JAVA_INT;
import static java.lang.foreign.ValueLayout.JAVA_LONG;

import java.lang.foreign.Arena;
import java.lang.foreign.MemorySegment;
import java.lang.ref.Cleaner;
import java.util.List;
import java.util.Queue;
import java.util.concurrent.ConcurrentLinkedQueue;
import java.util.concurrent.atomic.AtomicBoolean;

/**
 * The quantized matrices of a layer of experts and their products (j4q_experts_*); gate and up [experts * ffn, dim], down
 * [experts * dim, ffn]. Engine-local: the reference has no experts. Addresses are device addresses as
 * {@link Mi355xBackend#devicePointer} gives them, and the caller keeps what they belong to reachable until a sync; calls enqueue
 * on the engine stream and do not wait.
 *
 * <p>Holds its matrices, which the engine does not release before {@link #close()}; unreachable experts are destroyed on the
 * backend's next call, before any queued buffer release.
 */
public final class Mi355xExperts implements AutoCloseable {
  private static final Cleaner CLEANER = Cleaner.create();
  private static final Queue<Long> PENDING = new ConcurrentLinkedQueue<>();

  /** What lies between gate's product and up's (enum j4q_activation); GELU in its tanh form. */
  public enum Activation { SILU, GELU, RELU }

  /**
   * A norm of rows (j4q_norm): RMS, or with `layer` less the mean; weight and bias (device, fp32 [dim]; 0: ones, zeros);
   * weightAdd is added to the weights.
   */
  public record Norm(boolean layer, float eps, long weight, long bias, float weightAdd) {
    MemorySegment segment(Arena a) {
      MemorySegment s = a.allocate(32, 8);
      s.set(JAVA_INT, 0, layer ? Mi355xNative.NORM_LAYER : Mi355xNative.NORM_RMS);
      s.set(JAVA_FLOAT, 4, eps);
      s.set(JAVA_LONG, 8, weight);
      s.set(JAVA_LONG, 16, bias);
      s.set(JAVA_FLOAT, 24, weightAdd);
      return s;
    }
  }

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

  @SuppressWarnings({"unused", "FieldCanBeLocal"})
  private final List<Mi355xBuffer> matrices;  // kept reachable while the experts live
  private final State state;
  private final Cleaner.Cleanable cleanable;

  Mi355xExperts(long handle, List<Mi355xBuffer> matrices) {
    this.matrices = List.copyOf(matrices);
    this.state = new State(handle);
    this.cleanable = CLEANER.register(this, state);
  }

  /** j4q_experts_config. */
  static MemorySegment config(Arena a, long gate, long up, long down, int experts, Activation activation) {
    MemorySegment s = a.allocate(32, 8);
    s.set(JAVA_LONG, 0, gate);
    s.set(JAVA_LONG, 8, up);
    s.set(JAVA_LONG, 16, down);
    s.set(JAVA_INT, 24, experts);
    s.set(JAVA_INT, 28, activation.ordinal());
    return s;
  }

  /**
   * out[r] = sum over slots of weights[r, s] * down_e (act(gate_e x[r]) * (up_e x[r])), e = ids[r, s], none where that is no
   * expert's index; x and out F32 [rows, dim], strides in values (0: dense), ids int32 and weights F32 [rows, topK].
   */
  public void apply(long x, long xStride, long ids, long weights, long out, long outStride, long rows, int topK) {
    apply(x, xStride, ids, weights, out, outStride, rows, topK, Mi355xNative.KIND_F32);
  }

  /**
   * The same with bf16 x and out, as prompts have them: a third of the matrix instructions. The norm that adds its result takes it
   * as a bf16 block ({@link Mi355xBackend#norm} with blockBf16).
   */
  public void applyBf16(long x, long xStride, long ids, long weights, long out, long outStride, long rows, int topK) {
    apply(x, xStride, ids, weights, out, outStride, rows, topK, Mi355xNative.KIND_BF16);
  }

  private void apply(long x, long xStride, long ids, long weights, long out, long outStride, long rows, int topK, int type) {
    if (state.closed.get()) throw new IllegalStateException("experts are closed");
    try (Arena a = Arena.ofConfined()) {
      MemorySegment s = a.allocate(80, 8);  // without a workspace of the caller's
      s.set(JAVA_LONG, 0, x);
      s.set(JAVA_LONG, 8, ids);
      s.set(JAVA_LONG, 16, weights);
      s.set(JAVA_LONG, 24, out);
      s.set(JAVA_LONG, 32, rows);
      s.set(JAVA_LONG, 40, xStride);
      s.set(JAVA_LONG, 48, outStride);
      s.set(JAVA_INT, 56, topK);
      s.set(JAVA_INT, 60, type);
      Mi355xNative.call("expertsApply", Mi355xNative.EXPERTS_APPLY, state.handle, s, MemorySegment.NULL);
    }
  }

  /** Waits for the device, then destroys the handle; the matrices stay. Idempotent. */
  @Override
  public void close() {
    if (!state.closed.compareAndSet(false, true)) return;
    Mi355xNative.call("expertsDestroy", Mi355xNative.EXPERTS_DESTROY, state.handle);
    cleanable.clean();
  }

  static void drainPending() {
    for (Long h; (h = PENDING.poll()) != null; ) {
      try {
        Mi355xNative.status("expertsDestroy", Mi355xNative.EXPERTS_DESTROY, h.longValue());
      } catch (RuntimeException ignored) {
        // the library is gone: nothing to free
      }
    }
  }
}

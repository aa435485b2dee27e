/*
 * ilgpu_hip_algorithms.h — C ABI of libilgpu_hip_algorithms.so
 *
 * Hand-written gfx950 (MI355X, CDNA4) implementation of the data-parallel
 * primitives of ILGPU.Algorithms: radix sort (keys, key/value pairs), inclusive
 * and exclusive scan, reduction and histogram; and operators of language models
 * built beside them (embedding, layer norm, gradient norm and clipping).  The
 * entry points below are what a P/Invoke layer behind ILGPU's existing C#
 * surface binds; each primitive names the reference interface it stands in for
 * (paths relative to the ILGPU source tree).
 *
 * Conventions
 *  - Every pointer named keys/values/in/out/bins/overflow/temp is a DEVICE
 *    pointer to memory the caller owns (the address an ArrayView yields from
 *    LoadEffectiveAddressAsPtr, ArrayViewExtensions.cs:48-50).
 *  - `stream` is a hipStream_t (NULL = the default stream).  All work is
 *    enqueued asynchronously on it, like the reference's delegates; the
 *    caller synchronises before reading results.
 *  - Lengths and strides count ELEMENTS: element i of a view is at
 *    base[i * stride] (ArrayView1D<T, Stride1D.General>, ArrayViews.tt:114-119;
 *    Stride1D.Dense is stride 1).  Stride 1 takes the vectorised kernels;
 *    larger strides are served by scalar loads and stores (scan, reduce,
 *    histogram) or by a dense staging copy in temp (sort), and elements
 *    between the strided ones are never read or written.  Strides below 1
 *    return ILGPU_HIP_ERROR_OUT_OF_RANGE.
 *  - Lengths above INT32_MAX return ILGPU_HIP_ERROR_NOT_SUPPORTED, like
 *    ErrorMessages.NotSupportedArrayView64 in the reference.
 *  - The library allocates no device memory and keeps no pointer after a call
 *    returns.  Scratch space comes from `temp` (the reference's
 *    ArrayView<int> temp), sized by the *_temp_bytes queries; its contents on
 *    entry are irrelevant and on exit undefined.  One in-flight call per temp
 *    buffer; calls on different streams with different temps may overlap.
 *  - Return value: ilgpu_hip_status (0 = success).  Argument errors are
 *    detected before any GPU work is enqueued.
 */
#ifndef ILGPU_HIP_ALGORITHMS_H
#define ILGPU_HIP_ALGORITHMS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ILGPU_HIP_ALGORITHMS_VERSION 100 /* major*10000 + minor*100 + patch */

typedef void *ilgpu_hip_stream_t; /* hipStream_t */

/* Status codes and the .NET exception each maps to in the C# layer. */
typedef enum ilgpu_hip_status {
  ILGPU_HIP_SUCCESS = 0,
  ILGPU_HIP_ERROR_NULL_VIEW = 1,      /* ArgumentNullException: invalid view */
  ILGPU_HIP_ERROR_OUT_OF_RANGE = 2,   /* ArgumentOutOfRangeException */
  ILGPU_HIP_ERROR_NOT_SUPPORTED = 3,  /* NotSupportedException */
  ILGPU_HIP_ERROR_UNALIGNED_TEMP = 4, /* InvalidOperationException
                                         (TempViewManager.cs:98-106) */
  ILGPU_HIP_ERROR_RUNTIME = 5,        /* a HIP call failed; see
                                         ilgpu_hip_last_runtime_error() */
  ILGPU_HIP_ERROR_STATIC_LIMIT = 6    /* NotSupportedException: the input is
                                         larger than the library's static
                                         scratch serves (ilgpu_hip_scan_static) */
} ilgpu_hip_status;

/* Element types: NumericTypes of TypeInformation.ttinclude:94-121.  BF16 (the
 * upper half of a float32) has no counterpart there; only the operators at the
 * end of this header take it, the primitives answer NOT_SUPPORTED. */
typedef enum ilgpu_hip_type {
  ILGPU_HIP_I8 = 0, ILGPU_HIP_I16 = 1, ILGPU_HIP_I32 = 2, ILGPU_HIP_I64 = 3,
  ILGPU_HIP_U8 = 4, ILGPU_HIP_U16 = 5, ILGPU_HIP_U32 = 6, ILGPU_HIP_U64 = 7,
  ILGPU_HIP_F16 = 8, ILGPU_HIP_F32 = 9, ILGPU_HIP_F64 = 10,
  ILGPU_HIP_BF16 = 11
} ilgpu_hip_type;

/* Scan/reduce functors: Add/Max/Min of ScanReduceOperations.tt:20-27. */
typedef enum ilgpu_hip_op {
  ILGPU_HIP_OP_ADD = 0, ILGPU_HIP_OP_MAX = 1, ILGPU_HIP_OP_MIN = 2
} ilgpu_hip_op;

/* ScanKind (ScanExtensions.cs:27-38). */
typedef enum ilgpu_hip_scan_kind {
  ILGPU_HIP_SCAN_INCLUSIVE = 0, ILGPU_HIP_SCAN_EXCLUSIVE = 1
} ilgpu_hip_scan_kind;

/* Sort flags.  DESCENDING selects the Descending* functor
 * (RadixSortOperations.tt:98-125).  By default floating-point keys are
 * ordered exactly as the reference's ExtractRadixBits orders them
 * (RadixSortOperations.tt:81-89), and that order is NOT numerically monotone:
 * the mask meant to complement negative values comes from a logical shift of
 * an unsigned pattern, so an "ascending" sort of float or double keys leaves
 * the negative ones in ascending magnitude ([-0.5, -1, -2, 0.5, 1, 2]) and
 * positive keys that differ only in the last mantissa bit swapped; for Half
 * (whose bits are promoted to a 32-bit int before the shift) the negative
 * keys are in numeric order and the positive ones in descending order
 * ([-2, -1, -0.5, 2, 1, 0.5]).  FLOAT_TOTAL_ORDER instead sorts in IEEE-754
 * totalOrder (-NaN < -inf < ... < -0 < +0 < ... < +inf < +NaN), the
 * numerically sorted result; it has no counterpart in the reference. */
enum {
  ILGPU_HIP_SORT_DESCENDING = 1,
  ILGPU_HIP_SORT_FLOAT_TOTAL_ORDER = 2
};

/* Where the values of a key/value sort come from: the values view itself
 * (ViewSourceSequencer, Sequencer.cs:79-102) or value[i] = (TValue)i computed
 * on the fly.  FROM_INDEX: TValue is the integer type as wide as the value
 * (IndexSequencer, Sequencer.cs:36-45, and Int8Sequencer .. UInt64Sequencer,
 * Sequencers.tt:25-37: the index truncated to 1, 2, 4 or 8 bytes).
 * FROM_INDEX_AS_FLOAT: TValue is the floating-point type as wide as the value
 * (HalfSequencer, FloatSequencer, DoubleSequencer, Sequencer.cs:47-75: 2, 4 or
 * 8 bytes; long to float rounds to nearest even, Half goes through float as
 * the C# conversion does, so indices from 65520 on give +infinity). */
typedef enum ilgpu_hip_value_source {
  ILGPU_HIP_VALUES_FROM_VIEW = 0,
  ILGPU_HIP_VALUES_FROM_INDEX = 1,
  ILGPU_HIP_VALUES_FROM_INDEX_AS_FLOAT = 2
} ilgpu_hip_value_source;

/* Histogram bin locators (IComputeSingleBinOperation, IHistogramOperations.cs:
 * 19-30, is arbitrary user code in the reference; a native library offers a
 * closed set).  IDENTITY: bin = (int)value, elements outside [0, num_bins)
 * are ignored.  MODULO: bin = |value % num_bins|, the locator of the
 * reference's own tests (HistogramTests.tt:83-94). */
typedef enum ilgpu_hip_locator {
  ILGPU_HIP_LOCATOR_IDENTITY = 0,
  ILGPU_HIP_LOCATOR_MODULO = 1
} ilgpu_hip_locator;

/* ---- library ----------------------------------------------------------- */

int32_t ilgpu_hip_version(void);
const char *ilgpu_hip_status_string(int32_t status);
/* hipError_t of the most recent failing HIP call on the calling thread. */
int32_t ilgpu_hip_last_runtime_error(void);

/* Per-kernel timing, the library's counterpart of ILGPU's profiling markers
 * (ProfilingMarker.cs:19-61, enabled by Context.Builder.Profiling(),
 * Context.Builder.cs:315-319).  While enabled, each kernel launch is bracketed
 * by a pair of HIP events on its stream.  Enabling clears earlier totals.
 * ilgpu_hip_profile_query waits for the recorded events and returns how often
 * the named kernel ran and its summed duration.  Kernel names: "zero_words",
 * "reduce_partials", "reduce_final", "scan", "histogram", "sort_histogram",
 * "sort_plan", "sort_onesweep", "sort_finish".  Not meant for concurrent use
 * from several threads. */
int32_t ilgpu_hip_profile_enable(int32_t enabled);
int32_t ilgpu_hip_profile_query(const char *kernel_name, int64_t *launches,
                                double *total_ms);

/* ---- radix sort ---------------------------------------------------------
 * Replaces: RadixSort<T,TStride> delegates made by CreateRadixSort
 * (RadixSortExtensions.cs:37-42, 1130-1337), RadixSortPairs delegates made by
 * CreateRadixSortPairs (:56-96, 1017-1118) and the sizing helpers
 * ComputeRadixSortTempStorageSize / ComputeRadixSortPairsTempStorageSize
 * (:384-447).  Sorting is in place and stable; a pairs sort permutes `values`
 * with the keys.
 */

/* Bytes of temp needed to sort n keys of key_type, each with a payload of
 * value_bytes bytes (0 for a keys-only sort).  64-bit arithmetic throughout
 * (the reference's pair sizing multiplies in 32 bits). */
int32_t ilgpu_hip_radix_sort_temp_bytes(int64_t n, int32_t key_type,
                                        int32_t value_bytes,
                                        int64_t *temp_bytes);

/* The same for views with element strides above one: each strided view adds a
 * dense staging copy of its n elements.  ComputeRadixSortTempStorageSize has no
 * stride argument (RadixSortExtensions.cs:419-447: the reference's kernels
 * index through the view), so a binding offers this as an overload that takes
 * the views' strides; sorting a strided view with the dense size returns
 * ILGPU_HIP_ERROR_OUT_OF_RANGE (temp too small). */
int32_t ilgpu_hip_radix_sort_temp_bytes_strided(int64_t n, int32_t key_type,
                                                int32_t value_bytes,
                                                int64_t key_stride,
                                                int64_t value_stride,
                                                int64_t *temp_bytes);

int32_t ilgpu_hip_radix_sort_keys(ilgpu_hip_stream_t stream, void *keys,
                                  int64_t n, int64_t stride, int32_t key_type,
                                  int32_t flags, void *temp,
                                  int64_t temp_bytes);

/* value_bytes in {1, 2, 4, 8, 16}.  With ILGPU_HIP_VALUES_FROM_INDEX (value_bytes
 * 1, 2, 4 or 8) and ILGPU_HIP_VALUES_FROM_INDEX_AS_FLOAT (2, 4 or 8) the incoming
 * contents of `values` are ignored. */
int32_t ilgpu_hip_radix_sort_pairs(ilgpu_hip_stream_t stream, void *keys,
                                   int64_t key_stride, void *values,
                                   int64_t value_stride, int64_t n,
                                   int32_t key_type, int32_t value_bytes,
                                   int32_t flags, int32_t value_source,
                                   void *temp, int64_t temp_bytes);

/* How many 8-bit passes the last sort that used `temp` ran and how many it
 * found unnecessary (a pass whose digit is the same for every key is skipped:
 * keys below 2^16 run two passes of four, equal keys none; so are the lower digits that are
 * sorted after the passes, where few keys share the topmost ones: random keys of 4 and 8
 * bytes run one pass or two, and four of eight from 2^21 to 2^23 8-byte keys).  Same n, key_type
 * and value_bytes (0 for keys only) as that sort, dense views; waits for
 * `stream`.  The reference runs all NumBits / 2 passes whatever the keys
 * (RadixSortExtensions.cs:1276-1334) and has nothing to report. */
int32_t ilgpu_hip_radix_sort_passes(ilgpu_hip_stream_t stream, const void *temp,
                                    int64_t temp_bytes, int64_t n,
                                    int32_t key_type, int32_t value_bytes,
                                    int32_t *executed, int32_t *skipped);

/* Device self-check of the one hardware property the sort's ranking relies
 * on beyond the programming model: the lanes of ONE returning LDS atomic
 * instruction that meet in one address are served in ascending lane order
 * (this is what makes a pass stable at one LDS operation per key).  It has no
 * counterpart in the reference; its place there is taken by the group-wide
 * scans of RadixSortKernel1 (RadixSortExtensions.cs:700-705).  Plays `rows`
 * (1 .. 2^20) ranking rows per wave on every compute unit for six digit
 * distributions and stores the number of lanes found out of order in
 * mismatches[0] (device memory, 8-byte aligned): 0 on gfx950.  Stream-ordered,
 * allocates nothing. */
int32_t ilgpu_hip_selftest_lds_atomic_order(ilgpu_hip_stream_t stream,
                                            int32_t rows, int64_t *mismatches);

/* The same check, once per device and with the answer kept by the library:
 * ILGPU_HIP_SUCCESS for a device whose LDS serves the lanes in order,
 * ILGPU_HIP_ERROR_NOT_SUPPORTED for one that does not.  Every sort entry point
 * calls it first, so no sort runs on a device that has not passed: the first
 * sort on a device plays the check kernels (64 rows) on a counter inside the
 * library (nothing is allocated) and waits for `stream` once; later calls cost
 * one atomic load.  A stream that is being captured cannot be waited for: on a
 * device that has not been asked yet, a sort on such a stream (and this call)
 * returns ILGPU_HIP_ERROR_NOT_SUPPORTED, so callers that capture call this
 * first, outside the capture; accelerator objects of the host layers call it
 * in their constructors.  No counterpart in the reference. */
int32_t ilgpu_hip_sort_check_device(ilgpu_hip_stream_t stream);

/* TEST HOOK, not part of the product surface: process-wide parameters of the
 * sort for the library's own tests and tuning runs.  They are global mutable
 * state (a thread that changes one changes every sort of the process that is
 * launched afterwards), so applications leave them alone and bindings keep
 * them out of their public surface.  A negative value restores the default;
 * none has a counterpart in the reference (its passes are separate kernel
 * launches, RadixSortExtensions.cs:1276-1334).
 *   LOOKBACK_SPIN_LIMIT  how often the look-back of a pass polls the status
 *     word of an earlier tile that has published nothing before it stops
 *     waiting and counts that tile's digit itself from the source keys (tiles
 *     are handed to fixed groups of blocks, so a tile may wait for one whose
 *     group has no resident block; with this bound every block finishes
 *     whatever the others do).  A scan into another view takes the same bound
 *     and folds the tile from the input.  Default 4096; 0 makes every look-back
 *     that meets an empty word take the slow path at once, which is how the
 *     tests exercise it.
 *   LARGE_BLOCK_MIN_TILES_PER_CU  inputs of at least this many 1024-thread
 *     tiles per compute unit are sorted with 1024-thread blocks (longer runs
 *     per digit), smaller ones with 512-thread blocks (more blocks for fewer
 *     keys).  Default 3 for keys, 2 for pairs; 0 = always the large block,
 *     INT32_MAX = never.
 *   ONE_TILE_KERNEL  inputs of at most one 512-thread tile (18432 keys of up
 *     to 4 bytes, fewer for wider keys and for pairs) are sorted by one block
 *     in one launch, without temp memory.  Default 1; 0 sends them through
 *     the passes like longer inputs.
 *   ASSUME_LDS_ATOMIC_ORDER  what ilgpu_hip_sort_check_device answers: 0 = every
 *     device is taken to have failed the check (sorts return
 *     ILGPU_HIP_ERROR_NOT_SUPPORTED before anything is launched), 1 = taken to
 *     have passed, negative (the default) = the devices are asked, anew.
 *   SHORT_TILE_MAX_TILES  keys without values are cut into 512-thread tiles of
 *     a third, a half or two thirds of the usual length (6144, 9216 or 12288
 *     keys of up to 4 bytes), the shortest that makes at most this many tiles:
 *     more compute units at work on a short input.  Default 512, which is also
 *     the most that is taken (temp sizes assume it), and never more than two
 *     per compute unit; 0 = never. */
enum {
  ILGPU_HIP_SORT_PARAM_LOOKBACK_SPIN_LIMIT = 0,
  ILGPU_HIP_SORT_PARAM_LARGE_BLOCK_MIN_TILES_PER_CU = 1,
  ILGPU_HIP_SORT_PARAM_ONE_TILE_KERNEL = 2,
  ILGPU_HIP_SORT_PARAM_ASSUME_LDS_ATOMIC_ORDER = 3,
  ILGPU_HIP_SORT_PARAM_SHORT_TILE_MAX_TILES = 4
};
int32_t ilgpu_hip_sort_set_parameter(int32_t parameter, int32_t value);

/* ---- scan ---------------------------------------------------------------
 * Replaces: Scan<T,TStrideIn,TStrideOut> delegates made by CreateScan(kind)
 * (ScanExtensions.cs:52-61, 930-959) and ComputeScanTempStorageSize (:158-170).
 * elem_type in {I32, I64, U32, U64, F32, F64}.  out_length may exceed
 * in_length (only the first in_length outputs are written, :679-680);
 * shorter is ILGPU_HIP_ERROR_OUT_OF_RANGE.  in and out must not overlap
 * unless they are identical.
 */
int32_t ilgpu_hip_scan_temp_bytes(int64_t n, int32_t elem_type,
                                  int64_t *temp_bytes);

int32_t ilgpu_hip_scan(ilgpu_hip_stream_t stream, const void *in,
                       int64_t in_length, int64_t in_stride, void *out,
                       int64_t out_length, int64_t out_stride,
                       int32_t elem_type, int32_t op, int32_t kind, void *temp,
                       int64_t temp_bytes);

/* The same scan without a temp view, for callers that cannot allocate device
 * memory or carry a temp buffer: code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc.  It has no counterpart in the
 * reference (whose Scan delegates always take an ArrayView<int> temp,
 * ScanExtensions.cs:52-61).  The tile states live in a device array inside the
 * library (1 MiB + 256 bytes per GPU, held until the process ends), so
 *  - the input may hold at most ILGPU_HIP_SCAN_STATIC_MAX_BYTES bytes
 *    (in_length * element size); more returns ILGPU_HIP_ERROR_STATIC_LIMIT;
 *  - every call on one GPU uses that GPU's array: calls that overlap in time on
 *    the same GPU (two streams, two threads) race and must be serialised by the
 *    caller;
 *  - the call allocates nothing and clears what it needs with a fill kernel
 *    (no memset node), so it may be captured into a graph; the first call on a
 *    device looks up the array's address and should be made outside a capture.
 * Arguments, checks and results are those of ilgpu_hip_scan. */
#define ILGPU_HIP_SCAN_STATIC_MAX_BYTES (1ll << 30)
int32_t ilgpu_hip_scan_static(ilgpu_hip_stream_t stream, const void *in,
                              int64_t in_length, int64_t in_stride, void *out,
                              int64_t out_length, int64_t out_stride,
                              int32_t elem_type, int32_t op, int32_t kind);

/* ---- reduce -------------------------------------------------------------
 * Replaces: Reduction<T,TStride> delegates made by CreateReduction and the
 * Reduce overloads (ReductionExtensions.cs:30-35, 135-216).  out[0] is
 * overwritten with the fold of all inputs (:158-159); out_length >= 1.
 * Integer results are exact (wrapping adds); floating-point Add accumulates
 * in float64 in a fixed order, so repeated calls give identical bits.
 * The reference's delegate has no temp argument: the P/Invoke layer owns a
 * small scratch buffer of ilgpu_hip_reduce_temp_bytes() per delegate.
 */
int32_t ilgpu_hip_reduce_temp_bytes(int64_t n, int32_t elem_type,
                                    int64_t *temp_bytes);

int32_t ilgpu_hip_reduce(ilgpu_hip_stream_t stream, const void *in,
                         int64_t n, int64_t stride, int32_t elem_type,
                         int32_t op, void *out, int64_t out_length, void *temp,
                         int64_t temp_bytes);

/* ---- histogram ----------------------------------------------------------
 * Replaces: Histogram / HistogramUnchecked delegates and launchers
 * (HistogramExtensions.cs:35-59, 293-508; HistogramLaunchers.tt:52-101).
 * bins[locator(v)] += 1 for every input element; bins are ACCUMULATED into,
 * never cleared.  bin_type in {I32, I64, U32, U64, F32, F64}: the reference's
 * AtomicNumericTypes.  A floating-point bin receives its additions of 1.0 one
 * by one in its own precision, as Atomic.Add does, so a float bin stops
 * growing at 2^24 (16777216 + 1 rounds back to 16777216); the result is
 * computed exactly and does not depend on the order of the elements.  If
 * `overflow` is not NULL, overflow[0] |= 1 when some bin's count passed the
 * bin type's MaxValue (an increment found the bin holding MaxValue,
 * HistogramOperations.tt:36-40); NULL selects the unchecked variant.
 * in_type: any ilgpu_hip_type except F16.
 * Floating-point bins must live in ordinary device memory (hipMalloc: coarse
 * grained).  The counts of a block, and with more bins than LDS holds single
 * increments, go through the hardware's floating-point atomic add in L2, which
 * is exact there; for fine-grained, host-mapped or managed memory the hardware
 * does not promise that, and no reference fixture covers floating-point bins
 * at all.
 */
int32_t ilgpu_hip_histogram(ilgpu_hip_stream_t stream, const void *in,
                            int64_t n, int64_t stride, int32_t in_type,
                            void *bins, int64_t num_bins, int32_t bin_type,
                            int32_t locator, int32_t *overflow);

/* ---- unique -------------------------------------------------------------
 * Replaces: the Unique<T> delegate made by CreateUnique<T, Comparison<T>>, the
 * value-returning Unique and ComputeUniqueTempStorageSize
 * (UniqueExtensions.cs:27-33, 116-209).  Removes consecutive duplicates of
 * input[0..n) in place and writes the new length to new_length[0] (a device
 * int64, the reference's ArrayView<long> output).  Two elements are duplicates
 * if Comparison<T>.Compare yields 0 (ComparisonOperations.tt:30-45): CompareTo,
 * so all NaNs are equal and -0.0 equals +0.0.  elem_type: any of the eleven
 * numeric types.
 */
int32_t ilgpu_hip_unique_temp_bytes(int64_t n, int32_t elem_type,
                                    int64_t *temp_bytes);
int32_t ilgpu_hip_unique(ilgpu_hip_stream_t stream, void *input, int64_t n,
                         int32_t elem_type, int64_t *new_length,
                         int64_t new_length_extent, void *temp,
                         int64_t temp_bytes);

/* ---- initialize, sequence, reorder ----------------------------------------
 * Replace: Initializer delegates and Initialize (InitializeExtensions.cs:26-31,
 * 116-176): view[i] = *value, `value` being a HOST pointer to elem_bytes bytes
 * (1, 2, 4, 8 or 16); the Sequencer, RepeatedSequencer, BatchedSequencer and
 * RepeatedBatchedSequencer delegates (SequenceExtensions.cs:31-123, 238-630)
 * for the identity sequencers (Sequencers.tt:25-37, IndexSequencer):
 * view[i] = (T)((i / batch_length) % sequence_length), where Sequence passes
 * sequence_length = n and batch_length = 1; and Reorder
 * (ReorderExtensions.cs:194-214): target[i] = source[order[i]] for
 * i < order_length, with the reference's checks order_length >= source_length
 * and target_length >= order_length.  Index values are not range-checked.
 */
int32_t ilgpu_hip_initialize(ilgpu_hip_stream_t stream, void *view, int64_t n,
                             int64_t stride, int32_t elem_bytes,
                             const void *value);
int32_t ilgpu_hip_sequence(ilgpu_hip_stream_t stream, void *view, int64_t n,
                           int64_t stride, int32_t elem_type,
                           int64_t sequence_length, int64_t batch_length);
int32_t ilgpu_hip_reorder(ilgpu_hip_stream_t stream, const void *source,
                          int64_t source_length, void *target,
                          int64_t target_length, const int32_t *order,
                          int64_t order_length, int32_t elem_bytes);

/* ---- transform, reorder-transform ----------------------------------------
 * Replace: the Transformer delegates, CreateTransformer and Transform
 * (TransformExtensions.cs:73-115, 255-506): target[i] = f(source[i]) for
 * i < source_length, with the reference's checks source_length >= 1 and
 * target_length >= source_length (:304-317); and ReorderTransformer,
 * CreateReorderTransformer and ReorderTransform (ReorderExtensions.cs:42-52,
 * 143-297): target[i] = f(source[order[i]]) for i < order_length, with the
 * checks of ilgpu_hip_reorder.
 *
 * The reference JIT-compiles any ITransformer<TSource, TTarget> struct
 * (TransformExtensions.cs:24-37).  Here the transformers are a closed set of
 * the form (TTarget)op((TSource)value): op is computed in the source type
 * (integers wrap, as unchecked C#), then converted to the target type by the
 * C# explicit numeric conversion (integers truncate or extend by the source's
 * sign; to and between floating-point types: round to nearest even).  The set
 * covers IdentityTransformer (:42-55) and every transformer of the reference's
 * tests (Generic/AlgorithmsTestData.tt:170-252).  Floating-point sources with
 * integer targets are ILGPU_HIP_ERROR_NOT_SUPPORTED (C# leaves that conversion
 * unspecified for NaN and out-of-range values), and so is BIT_COMPLEMENT of a
 * floating-point source.  `factor` is used by MULTIPLY only, converted to the
 * source type.  A transform with equal source and target types may run in
 * place (source == target, equal strides).
 */
enum ilgpu_hip_transformer {
  ILGPU_HIP_TRANSFORM_CONVERT = 0,        /* (TTarget)value; identity if the types match */
  ILGPU_HIP_TRANSFORM_NEGATE = 1,         /* (TTarget)(-value) */
  ILGPU_HIP_TRANSFORM_BIT_COMPLEMENT = 2, /* (TTarget)(~value), integer sources */
  ILGPU_HIP_TRANSFORM_MULTIPLY = 3        /* (TTarget)(value * (TSource)factor) */
};
int32_t ilgpu_hip_transform(ilgpu_hip_stream_t stream, const void *source,
                            int64_t source_length, int64_t source_stride,
                            int32_t source_type, void *target,
                            int64_t target_length, int64_t target_stride,
                            int32_t target_type, int32_t transformer,
                            int64_t factor);
int32_t ilgpu_hip_reorder_transform(ilgpu_hip_stream_t stream,
                                    const void *source, int64_t source_length,
                                    int32_t source_type, void *target,
                                    int64_t target_length, int32_t target_type,
                                    const int32_t *order, int64_t order_length,
                                    int32_t transformer, int64_t factor);

/* ---- operators of language models -------------------------------------------
 * No counterpart in the reference.  They follow the conventions above, and:
 *  - A matrix is given by its first element, its rows and columns and its row
 *    stride in elements; element (r, c) is at base[r * row_stride + c].  The
 *    row stride of a matrix that is read may be anything from 0 (one row for
 *    all); that of a matrix that is written is at least its columns
 *    (ILGPU_HIP_ERROR_OUT_OF_RANGE otherwise).  Any element-aligned base and any
 *    stride up to INT32_MAX, as of rows and columns, will do; rows need no
 *    alignment of their own.
 *  - Types are ILGPU_HIP_F32, F16 and BF16 (others: ILGPU_HIP_ERROR_NOT_SUPPORTED).
 *    All arithmetic is in float32 or wider; each result is rounded to its type
 *    once, to nearest even.
 *  - No rows, no tokens, no tensors are valid inputs: the call does what the
 *    formula says for an empty sum.  A null pointer is ILGPU_HIP_ERROR_NULL_VIEW
 *    where there is something to read or write; zero columns always are.
 *  - Single numbers (scale, epsilon, max_norm) are HOST pointers, read before
 *    the call returns.
 *  - Results do not depend on the order in which blocks run: the same call on
 *    the same inputs gives the same bits.
 */

/* Embedding: out[i] = scale * table[tokens[i]] for every i < count, rows of
 * `dimension` elements.  tokens: int32 or int64 (token_type).  A token outside
 * [0, vocabulary) gives a row of zeros and is never used as an address.
 * scale: NULL means 1.  Any of the three types for the table and for out. */
int32_t ilgpu_hip_embedding(ilgpu_hip_stream_t stream, const void *table,
                            int64_t vocabulary, int64_t dimension,
                            int64_t table_stride, int32_t table_type,
                            const void *tokens, int64_t count,
                            int32_t token_type, const float *scale, void *out,
                            int64_t out_stride, int32_t out_type);

/* Its gradient: grad_table[v] (+)= scale * sum of grad_out[i] over the positions
 * i with tokens[i] == v, added up in float32.  Every row of
 * grad_table is written, with zeros where no position has its token; with
 * accumulate != 0 the sums are added to what is there instead, and other rows
 * are left alone.  Tokens outside [0, vocabulary) and padding_token (pass -1
 * for none) contribute nothing.  grad_table must not overlap grad_out or
 * tokens.  On a device whose LDS fails ilgpu_hip_sort_check_device:
 * ILGPU_HIP_ERROR_NOT_SUPPORTED, like a sort.  A temp for `count` tokens serves
 * any smaller number of them (same vocabulary and dimension). */
int32_t ilgpu_hip_embedding_gradient_temp_bytes(int64_t count,
                                                int64_t vocabulary,
                                                int64_t dimension,
                                                int64_t *temp_bytes);
int32_t ilgpu_hip_embedding_gradient(
    ilgpu_hip_stream_t stream, const void *grad_out, int64_t grad_out_stride,
    int32_t grad_out_type, const void *tokens, int64_t count,
    int32_t token_type, const float *scale, int64_t padding_token,
    int32_t accumulate, void *grad_table, int64_t vocabulary,
    int64_t dimension, int64_t grad_table_stride, int32_t grad_table_type,
    void *temp, int64_t temp_bytes);

/* Layer norm of every row: out = (in - m) * r * weight + bias with m the row's
 * mean, r = 1 / sqrt(v + epsilon) and v the mean of (in - m)^2.  weight and bias
 * (`columns` elements of weight_type, which is `type` or F32) may be NULL: 1 and
 * 0.  mean and rstd (float32, one per row) receive m and r and may be NULL.
 * in and out have the same type; out may be in itself (same base and stride).
 * epsilon: finite and not negative.  Of a row whose mean is more than two
 * deviations from zero the mean is found in two steps, so that its size costs
 * out and rstd no bits.  Squared deviations are float32: a row with deviations
 * beyond 1e19 overflows (rstd 0), as one with an infinity is NaN. */
int32_t ilgpu_hip_layer_norm(ilgpu_hip_stream_t stream, const void *in,
                             int64_t rows, int64_t columns, int64_t in_stride,
                             int32_t type, const void *weight,
                             const void *bias, int32_t weight_type,
                             const float *epsilon, void *out,
                             int64_t out_stride, float *mean, float *rstd);

/* Its gradients from mean and rstd as the forward call left them: with
 * h = (in - mean) * rstd and g = weight * grad_out,
 *   grad_in     = rstd * (g - mean of g - h * mean of g * h)   (means over the row)
 *   grad_weight = sum over the rows of grad_out * h
 *   grad_bias   = sum over the rows of grad_out
 * (mean is a float32: where it is large against the row's deviations, its rounding
 * is in every h.)
 * weight may be NULL (1).  Each of grad_in, grad_weight and grad_bias may be NULL
 * and is not computed then; not all of them.  grad_in may be grad_out itself or in
 * itself (same base and stride).  With accumulate != 0 grad_weight and grad_bias
 * are added to what is there.  No rows leave sums of zero. */
int32_t ilgpu_hip_layer_norm_gradient_temp_bytes(int64_t rows, int64_t columns,
                                                 int64_t *temp_bytes);
int32_t ilgpu_hip_layer_norm_gradient(
    ilgpu_hip_stream_t stream, const void *grad_out, int64_t grad_out_stride,
    const void *in, int64_t in_stride, int64_t rows, int64_t columns,
    int32_t type, const void *weight, int32_t weight_type, const float *mean,
    const float *rstd, void *grad_in, int64_t grad_in_stride,
    void *grad_weight, void *grad_bias, int32_t accumulate, void *temp,
    int64_t temp_bytes);

/* One array of a list: `length` dense elements of `type` at `data`.  The list
 * itself is HOST memory, read before the call returns. */
typedef struct ilgpu_hip_tensor {
  void *data;
  int64_t length;
  int32_t type;
  int32_t reserved; /* 0 */
} ilgpu_hip_tensor;

/* norm[0] = the root of the sum of the squares of all elements of all tensors,
 * added up in float64.  At most 2^40 elements and INT32_MAX tensors (beyond:
 * ILGPU_HIP_ERROR_NOT_SUPPORTED); tensors of length 0 are skipped. */
int32_t ilgpu_hip_gradient_norm_temp_bytes(int64_t count, int64_t *temp_bytes);
int32_t ilgpu_hip_gradient_norm(ilgpu_hip_stream_t stream,
                                const ilgpu_hip_tensor *tensors, int64_t count,
                                float *norm, void *temp, int64_t temp_bytes);

/* targets[k] = factor * sources[k], element for element, with
 * factor = max_norm / norm[0] where norm[0] is finite and larger than max_norm,
 * 1 otherwise: an infinite or NaN norm leaves the values as they are, and norm[0]
 * tells.  norm is DEVICE memory (ilgpu_hip_gradient_norm's, or combined over
 * processes); nothing waits for it on the host.  targets[k] has the length and
 * type of sources[k] and is the same array or does not overlap any source; targets
 * NULL: in place.  Tensors that a factor of 1 leaves as they are in place are not
 * touched.  max_norm: not negative, not NaN. */
int32_t ilgpu_hip_clip_gradients(ilgpu_hip_stream_t stream,
                                 const ilgpu_hip_tensor *sources,
                                 const ilgpu_hip_tensor *targets,
                                 int64_t count, const float *norm,
                                 const float *max_norm);

/* Gated linear recurrence, one of its own in every channel (column):
 *   h[t] = a[t] * h[t-1] + b[t]
 * with a = 1 / (1 + exp(-gate)) or exp(gate) (decay) and b = in, or (1 - a) * in
 * with complement != 0; 1 - a keeps its precision where a is near 1.  out[t] is
 * h[t], rounded to `type`; the states themselves are float32 throughout.
 * Sequences lie behind one another in the rows: sequence i is rows
 * [offsets[i], offsets[i+1]) with offsets (sequences + 1 numbers, int32 or int64)
 * in DEVICE memory, or, with offsets NULL, the i-th of `sequences` equal parts
 * (rows must be a multiple: ILGPU_HIP_ERROR_OUT_OF_RANGE).  In front of its first
 * row a sequence has the state initial[i] (sequences x channels, float32; NULL:
 * zeros), behind its last it leaves final_state[i] (NULL: not wanted), and a
 * sequence without rows leaves what it began with.  Nothing passes from one
 * sequence to another, NaN and infinities neither.  Rows in front of the first
 * sequence and behind the last are not written.  offsets ascend from 0 or more to
 * at most rows; others give unspecified results, but no access outside the
 * matrices.
 * Decays and states are float32: exp(gate) of a gate above 88.7 is infinite, of one
 * below -87.3 it may be zero, and a state that decays above 1 take beyond the
 * largest float32 is infinite or a NaN from there on.  The decays of many rows may
 * leave float32 together, as long as the states do not.
 * One row for each sequence (offsets NULL, sequences == rows) is the step from
 * token to token; it needs no temp.
 * out may be gate or in itself, final_state may be initial itself (same base and
 * stride); otherwise what is written overlaps nothing.  A temp for so many rows
 * serves any fewer (same channels), and both directions; it may be NULL where the
 * size asked for is 0. */
enum ilgpu_hip_decay {
  ILGPU_HIP_DECAY_SIGMOID = 0,    /* a = 1 / (1 + exp(-gate)) */
  ILGPU_HIP_DECAY_EXPONENTIAL = 1 /* a = exp(gate) */
};
int32_t ilgpu_hip_gated_recurrence_temp_bytes(int64_t rows, int64_t channels,
                                              int64_t *temp_bytes);
int32_t ilgpu_hip_gated_recurrence(
    ilgpu_hip_stream_t stream, const void *gate, int64_t gate_stride,
    const void *in, int64_t in_stride, int64_t rows, int64_t channels,
    int32_t type, int32_t decay, int32_t complement, const void *offsets,
    int32_t offset_type, int64_t sequences, const float *initial,
    int64_t initial_stride, void *out, int64_t out_stride, float *final_state,
    int64_t final_stride, void *temp, int64_t temp_bytes);

/* Its gradients from those of out and of the final states (grad_final NULL:
 * zeros).  With G[t] = grad_out[t] + a[t+1] * G[t+1], the last G of a sequence
 * being its grad_out + grad_final:
 *   grad_in      = G, or (1 - a) * G with complement
 *   grad_gate    = G * (h[t-1], less in[t] with complement) * da
 *                  with da = a * (1 - a) or a
 *   grad_initial = a * G of the first row, or grad_final where there is none
 * h[t-1] is out as the forward call left it, or initial.  Each of grad_gate,
 * grad_in and grad_initial may be NULL and is not computed then; not all of them.
 * grad_gate and grad_in may be grad_out, gate or in itself, not both the same;
 * grad_initial may be grad_final itself. */
int32_t ilgpu_hip_gated_recurrence_gradient(
    ilgpu_hip_stream_t stream, const void *grad_out, int64_t grad_out_stride,
    const void *gate, int64_t gate_stride, const void *in, int64_t in_stride,
    const void *out, int64_t out_stride, int64_t rows, int64_t channels,
    int32_t type, int32_t decay, int32_t complement, const void *offsets,
    int32_t offset_type, int64_t sequences, const float *initial,
    int64_t initial_stride, const float *grad_final, int64_t grad_final_stride,
    void *grad_gate, int64_t grad_gate_stride, void *grad_in,
    int64_t grad_in_stride, float *grad_initial, int64_t grad_initial_stride,
    void *temp, int64_t temp_bytes);

/* What stands between two blocks of a model: the norm behind the one and its gate,
 * the residual stream with its scale, and the norm in front of the next.  For every
 * row, with rms(v) = 1 / sqrt(mean of v^2 + epsilon):
 *   y     = in [* input_rstd * input_weight] [* act(gate)]    input_rstd = rms(in)
 *   total = residual + scale * y
 *   out   = total * rstd * weight                             rstd = rms(total)
 * The input is normalised with input_norm != 0, and input_weight NULL is 1 then;
 * act(gate) is gate_kind's function of the matrix gate, or 1 where gate is NULL.
 * residual NULL: 0.  weight NULL: 1.  scale NULL: 1.  total and out may each be NULL
 * and are not written then; not both.  Weights have `columns` elements of
 * weight_type, which is `type` or F32; residual and total are of residual_type,
 * which is `type` or F32 too.  input_rstd and rstd (float32, one per row) receive
 * what the gradients need and may be NULL.  out is made from total before it is
 * rounded to its type.  total may be residual itself; out (and total, of the same
 * type) may be in or gate itself (same base and stride).  Squares are float32: rows beyond
 * 1e19 overflow. */
enum ilgpu_hip_gate {
  ILGPU_HIP_GATE_SIGMOID = 0, /* 1 / (1 + exp(-gate)) */
  ILGPU_HIP_GATE_SILU = 1     /* gate / (1 + exp(-gate)) */
};
int32_t ilgpu_hip_residual_norm(
    ilgpu_hip_stream_t stream, const void *in, int64_t in_stride, int64_t rows,
    int64_t columns, int32_t type, int32_t input_norm,
    const void *input_weight, const void *gate, int64_t gate_stride,
    int32_t gate_kind, const void *residual, int64_t residual_stride,
    int32_t residual_type, const float *scale, const void *weight,
    int32_t weight_type, const float *epsilon, void *total,
    int64_t total_stride, void *out, int64_t out_stride, float *input_rstd,
    float *rstd);

/* Its gradients from those of out (NULL: out was not used; then total, weight and
 * rstd are not either) and of total (NULL: only out was used); not both NULL.  total
 * and both rstd are the forward call's.  With h = total * rstd, g = grad_out * weight,
 * k = in * input_rstd:
 *   grad_residual     = grad_total + rstd * (g - h * mean of g * h)     =: d
 *   grad_weight       = sum over the rows of grad_out * h
 *   grad_gate         = scale * d * (k * input_weight) * act'(gate)
 *   grad_input_weight = sum over the rows of e * k       e = scale * d * act(gate)
 *   grad_in           = input_rstd * (f - k * mean of f * k)  f = e * input_weight
 * and without input_norm k * input_weight is in, and grad_in is e.  Each of the
 * five may be NULL and is not computed then; not all of them.
 * grad_in, grad_gate and grad_residual may be any of the matrices that are read
 * (of the same type; same base and stride), not the same one.  With accumulate != 0 grad_weight and
 * grad_input_weight are added to what is there.  No rows leave sums of zero.  A temp
 * for so many rows serves any fewer (same columns). */
int32_t ilgpu_hip_residual_norm_gradient_temp_bytes(int64_t rows,
                                                    int64_t columns,
                                                    int64_t *temp_bytes);
int32_t ilgpu_hip_residual_norm_gradient(
    ilgpu_hip_stream_t stream, const void *grad_out, int64_t grad_out_stride,
    const void *grad_total, int64_t grad_total_stride, const void *in,
    int64_t in_stride, int64_t rows, int64_t columns, int32_t type,
    int32_t input_norm, const void *input_weight, const float *input_rstd,
    const void *gate, int64_t gate_stride, int32_t gate_kind,
    const void *total, int64_t total_stride, int32_t residual_type,
    const float *scale, const void *weight, int32_t weight_type,
    const float *rstd, void *grad_in, int64_t grad_in_stride, void *grad_gate,
    int64_t grad_gate_stride, void *grad_residual,
    int64_t grad_residual_stride, void *grad_input_weight, void *grad_weight,
    int32_t accumulate, void *temp, int64_t temp_bytes);

/* One step of AdamW over lists of `count` tensors, in place: for every element
 *   g = f * gradient,  m = beta1 * m + (1 - beta1) * g,  v = beta2 * v + (1 - beta2) * g^2
 *   p = p - r * (m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + epsilon) + weight_decay * p)
 * t = step[0] (int64, DEVICE memory, 1 for the first step; the caller counts it on),
 * r = rate * schedule[0] (float32, DEVICE memory; NULL: 1), so that a captured step
 * goes on counting when it is replayed.  norm (float32, DEVICE memory, as
 * ilgpu_hip_gradient_norm leaves it; NULL: f = 1): f is max_norm / norm[0] where that
 * is less than 1, else 1; where norm[0] is infinite or NaN nothing at all is changed.
 * parameters[k], gradients[k] and copies[k] (copies NULL: none) have the same length
 * and each its type, F32, F16 or BF16; copies receive p too, rounded to their own
 * type.
 * Moments in 32 bits (first_scales and second_scales NULL): first[k] and second[k]
 * are F32 of the same length, zeros before the first step.
 * Moments in 8 bits: first[k] and second[k] are U8 of the same length, and
 * first_scales[k] and second_scales[k] F32 with one element for every 256 of it (the
 * last may stand for fewer), the largest |m| and v among them; all zeros before the first step.  A code c
 * of the first stands for s * q * |q| / 127^2 with q = c - 128, of the second for
 * s * c^4 / 255^4, s the scale.  p is computed from m and v before they are rounded.
 * They are rounded up or down so that they are right in the mean, which lets moments
 * move that change by less than a code's distance in a step: with u a number in
 * [0, 1) from a hash of (seed, t, k, index), the code below the value is raised by
 * one where the value is more than u of the way to the next.  (Where the largest of a
 * block is below 1e-27 the second moments lose digits, below the normal float32
 * numbers a block is stored as zeros; a gradient that is not finite, without a norm,
 * spoils the moments of its 256.)  m and v are made by products and sums rounded to
 * float32 one by one, so that codes are the same wherever they are computed so.
 * Nothing that is written overlaps anything else.  Tensors of length 0 are skipped. */
typedef struct ilgpu_hip_adamw_options {
  double rate;         /* not negative, finite */
  double beta1, beta2; /* [0, 1) */
  double epsilon;      /* a positive normal float32 */
  double weight_decay; /* not negative, finite */
  double max_norm;     /* not negative, not NaN; used with norm */
  int64_t seed;        /* of 8-bit moments */
} ilgpu_hip_adamw_options;
int32_t ilgpu_hip_adamw(ilgpu_hip_stream_t stream,
                        const ilgpu_hip_tensor *parameters,
                        const ilgpu_hip_tensor *gradients,
                        const ilgpu_hip_tensor *first,
                        const ilgpu_hip_tensor *second,
                        const ilgpu_hip_tensor *first_scales,
                        const ilgpu_hip_tensor *second_scales,
                        const ilgpu_hip_tensor *copies, int64_t count,
                        const ilgpu_hip_adamw_options *options,
                        const int64_t *step, const float *schedule,
                        const float *norm);

/* 8-bit moments as the numbers they stand for, into tensors of the same lengths
 * (F32, F16 or BF16).  first, first_scales and first_targets may be NULL together,
 * as may be the second's three; not all six. */
int32_t ilgpu_hip_adamw_moments(ilgpu_hip_stream_t stream,
                                const ilgpu_hip_tensor *first,
                                const ilgpu_hip_tensor *first_scales,
                                const ilgpu_hip_tensor *first_targets,
                                const ilgpu_hip_tensor *second,
                                const ilgpu_hip_tensor *second_scales,
                                const ilgpu_hip_tensor *second_targets,
                                int64_t count);

#ifdef __cplusplus
}
#endif
#endif /* ILGPU_HIP_ALGORITHMS_H */

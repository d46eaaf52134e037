/*
 * C ABI of libthundergbm.so (MI355X build).
 *
 * Part 1 is the drop-in boundary: the nine entry points that the reference's Python wrapper
 * (python/thundergbm/thundergbm.py) binds with ctypes, with the argument order, types and
 * ownership rules of src/thundergbm/scikit_tgbm.cpp, plus the two file-based entry points of the R
 * interface (src/thundergbm/gbm_R_interface.cpp). Where the reference declares `Tree *&model`
 * the ABI passes the address of an 8-byte slot; it is spelled `tgbm_model **` here. The model is
 * opaque, owned by the library and released only by model_free().
 *
 * Part 2 is a session API over the same trainer for callers that keep data resident in HBM between
 * calls (the benchmark) or drive the stages one by one (the parity tests).
 *
 * Failures abort the process after printing a FATAL line, as the reference's CHECK macros do.
 * One call trains on one GPU and blocks until done. The training and prediction calls of part 1 hold a
 * process-wide lock (the reference serialises Booster::boost with a global mutex, booster.h:17,78), so calls
 * from several threads run one after the other; a session of part 2 belongs to one thread at a time.
 */
#ifndef THUNDERGBM_H
#define THUNDERGBM_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct tgbm_model tgbm_model;

/* ---------------------------------------------------------------- Part 1: reference boundary */

/* scikit_tgbm.cpp:13-23. verbose 0 = silent, 1 = info, 2 = debug. */
void set_logger(int verbose);

/* scikit_tgbm.cpp:26-80. CSR input (float32 values, int32 indices, ascending columns per row).
 * num_class is in/out, group_label receives the distinct labels (caller allocates one float per
 * distinct label), tree_per_iter and *model are outputs. column_sampling_rate < 1 samples columns per
 * round as the reference does (see tgbm_trainer_set_option). group / num_group are the query group sizes
 * of the ranking objectives (rank:pairwise, rank:ndcg; dataset.cpp:64-68) and ignored otherwise. bagging != 0
 * resamples the gradients every round (RowSampler::do_bagging, row_sampler.cu:9-38, booster.h:84). n_device
 * and n_parallel_trees (never read by the reference either) are accepted for signature compatibility and
 * ignored. */
void sparse_train_scikit(int row_size, float *val, int *row_ptr, int *col_ptr, float *label, int depth, int n_trees,
                         int n_device, float min_child_weight, float lambda, float gamma, int max_num_bin,
                         int verbose, float column_sampling_rate, int bagging, int n_parallel_trees,
                         float learning_rate, char *obj_type, int *num_class, char *tree_method, tgbm_model **model,
                         int *tree_per_iter, float *group_label, int *group, int num_group);

/* sparse_train_scikit for a dense matrix x: float (x_is_double 0) or double [row_size][columns], row by row, fewer than
 * 2^32 cells. A zero is a value that is not stored, as for the reference's wrapper, which drops the zeros of dense input
 * on its way to CSR (thundergbm.py:98-103); doubles are trained on as floats. group_label has row_size slots, n_distinct
 * receives the number of distinct labels. The other arguments and the model are those of sparse_train_scikit on the same
 * data. It has no counterpart in the reference. */
void tgbm_train_dense(int row_size, int columns, const void *x, int x_is_double, const float *label, int depth,
                      int n_trees, int n_device, float min_child_weight, float lambda, float gamma, int max_num_bin,
                      int verbose, float column_sampling_rate, int bagging, int n_parallel_trees, float learning_rate,
                      const char *obj_type, int *num_class, const char *tree_method, tgbm_model **model,
                      int *tree_per_iter, float *group_label, int *n_distinct, const int *group, int num_group);

/* scikit_tgbm.cpp:83-121. y_pred: row_size floats, or row_size * num_class (class-major) for
 * multi:softprob. As in the reference the base score is not part of this path. group / num_group: query
 * groups of the rows for a ranking objective; they only feed the metric line of the log and may be absent. */
void sparse_predict_scikit(int row_size, float *val, int *row_ptr, int *col_ptr, float *y_pred, tgbm_model **model,
                           int n_trees, int trees_per_iter, char *objective, int num_class, float learning_rate,
                           float *group_label, int *group, int num_group, int verbose);

/* sparse_predict_scikit for a dense matrix (x, x_is_double: see tgbm_train_dense). The predictions are those of
 * sparse_predict_scikit on the same data. It has no counterpart in the reference. */
void tgbm_predict_dense(int row_size, int columns, const void *x, int x_is_double, float *y_pred, tgbm_model **model,
                        int n_trees, int trees_per_iter, const char *objective, int num_class, float learning_rate,
                        const float *group_label, const int *group, int num_group, int verbose);

/* scikit_tgbm.cpp:123-147 / parser.cpp:146-171: raw binary model file. */
void save(char *model_path, char *objective, float learning_rate, int num_class, int n_trees, int trees_per_iter,
          tgbm_model **model, float *group_label);

/* scikit_tgbm.cpp:148-172 / parser.cpp:102-145. */
void load_model(char *model_path, float *learning_rate, int *num_class, int *n_trees, int *trees_per_iter,
                tgbm_model **model);

/* scikit_tgbm.cpp:173-182: the label table of a model file. */
void load_config(char *model_path, float *group_label);

/* scikit_tgbm.cpp:184-197: node count of every tree (all 2^(depth+1)-1 heap slots). */
void get_n_nodes(tgbm_model **model, int *n_nodes, int n_trees, int tree_per_iter);

/* scikit_tgbm.cpp:199-248: one tree as parallel arrays in heap order. */
void get_a_tree(tgbm_model **model, int tree_id, int n_nodes, int *children_left, int *children_right,
                int *children_default, int *features, float *thresholds, float *values,
                float *node_sample_weights);

/* The first n_trees trees like that, one behind the other in every array (get_n_nodes tells how long each is). */
void tgbm_get_trees(tgbm_model **model, int n_trees, int *children_left, int *children_right, int *children_default, int *features,
                    float *thresholds, float *values, float *node_sample_weights);

/* scikit_tgbm.cpp:250-254. */
void model_free(tgbm_model **model);

/* gbm_R_interface.cpp:10-61 and :63-86, the two symbols R/gbm.R reaches with .C(): every argument is a
 * pointer, strings are char**. train_R loads the LIBSVM file data[0] (plus data[0].group for a ranking
 * objective), trains and writes the model file model_out[0]; predict_R loads model_in[0] and the file
 * data[0], predicts and logs the metric. min_child_weight is an int here, as in the reference. */
void train_R(int *depth, int *n_trees, int *n_gpus, int *verbose, int *profiling, char **data, int *max_num_bin,
             double *column_sampling_rate, int *bagging, int *n_parallel_trees, double *learning_rate,
             char **objective, int *num_class, int *min_child_weight, double *lambda_tgbm, double *gamma,
             char **tree_method, char **model_out);
void predict_R(char **data, char **model_in, int *verbose);

/* ------------------------------------------------------------------- Part 2: session API */

typedef struct tgbm_trainer tgbm_trainer;

/* DataSet::load_from_sparse + HistTreeBuilder_single::init + Booster::init
 * (dataset.cpp:20-63, hist_tree_builder_single.cu:783-844, booster.h:36-74): copies the CSR input
 * to the GPU, builds cut points, the bin matrix and the base score. */
tgbm_trainer *tgbm_trainer_create(int row_size, const float *val, const int *row_ptr, const int *col_ptr,
                                  const float *label, int depth, int n_trees, float min_child_weight, float lambda,
                                  float gamma, int max_num_bin, float learning_rate, const char *objective,
                                  int num_class, int verbose);
/* The same with query groups for the ranking objectives rank:pairwise / rank:ndcg (LambdaRank,
 * LambdaRankNDCG: objective/ranking_obj.cpp:11-18, :100-103): `group` holds num_group sizes of consecutive
 * runs of rows that sum to row_size, as in the group / num_group arguments of sparse_train_scikit
 * (scikit_tgbm.cpp:31, dataset.cpp:64-68). Other objectives ignore them. */
tgbm_trainer *tgbm_trainer_create_grouped(int row_size, const float *val, const int *row_ptr, const int *col_ptr,
                                          const float *label, int depth, int n_trees, float min_child_weight,
                                          float lambda, float gamma, int max_num_bin, float learning_rate,
                                          const char *objective, int num_class, int verbose, const int *group,
                                          int num_group);
void tgbm_trainer_destroy(tgbm_trainer *t);

/* Options that tgbm_trainer_create has no argument for. "column_sampling_rate" (GBMParam, common.h:92):
 * below 1 every boosting round ignores max(1, int(n_features * rate)) randomly chosen columns in its split
 * search (Shard::column_sampling, builder/shard.cu:8-22; the shuffle draws from the process-wide rand()).
 * "bagging" (common.h:97): non-zero makes every gradient pass multiply the gradient pairs by bootstrap draw
 * counts (RowSampler::do_bagging, row_sampler.cu:9-38; seeded with one rand() per pass).
 * "reorder_first", "reorder_burst", "reorder_every", "reorder_min_rows" (no counterpart in the reference):
 * tgbm_trainer_boost physically re-orders the rows by the leaves of the tree just built after each of the
 * trees `reorder_first` .. `reorder_first + reorder_burst - 1` and then every `reorder_every` trees
 * (defaults 1, 3 and 32; reorder_first 0 = never) when the dataset has at least
 * `reorder_min_rows` rows (default 2^20), the layout is dense and the objective is not a ranking one. Results do not
 * depend on it beyond float round-off, and all per-row buffers keep the caller's row order. */
void tgbm_trainer_set_option(tgbm_trainer *t, const char *key, double value);
/* The column sampling of one round for stage-wise driving (tgbm_trainer_boost does it itself). */
void tgbm_trainer_sample_columns(tgbm_trainer *t);

/* `rounds` iterations of Booster::boost (booster.h:76-93); returns after the GPU finished. */
void tgbm_trainer_boost(tgbm_trainer *t, int rounds);

/* Stage-wise driving; each call returns after enqueueing (tgbm_trainer_get synchronises).
 * gradient = ObjectiveFunction::get_gradient (then do_bagging when the option is on); tree_init = Tree::init2; find_split = find_split +
 * update_tree of the level; partition = update_ins2node_id; finish_tree = prune_self +
 * predict_in_training. */
void tgbm_trainer_gradient(tgbm_trainer *t);
void tgbm_trainer_tree_init(tgbm_trainer *t, int class_id);
void tgbm_trainer_find_split(tgbm_trainer *t, int level);
void tgbm_trainer_partition(tgbm_trainer *t, int level);
void tgbm_trainer_finish_tree(tgbm_trainer *t, int class_id);
float tgbm_trainer_metric(tgbm_trainer *t);

/* Integer facts: n, n_features, n_bins, num_class, tree_per_rounds, n_nodes, dense_W,
 * dense_blocks, dense_cols (columns of the dense bin matrix: fewer than n_features when runs of features
 * that never meet in a row share a column), trees_built, rounds_done, n_packs, depth, y_pred_size, max_hitems, n_sets (class trees
 * of a round built by common launches), reorders_done, device_free_mb (free device memory in MiB). */
int tgbm_trainer_info(tgbm_trainer *t, const char *key);
float tgbm_trainer_base_score(tgbm_trainer *t);

/* Copies a device buffer to `out` when `cap` is large enough; always returns its size in bytes.
 * Names: cut_val, cut_row_ptr, cut_fid, binmat (dense layout: [dense_blocks][n][dense_W] bins of the matrix's
 * columns; with dense_cols < n_features feature f is column feat_col[f] and its local bin b is stored as
 * feat_lo[f] + b), feat_col (int per feature), feat_lo (byte per feature), nid, gh, y_pred, y, nodes, sp, hist_q0, hist_q1,
 * quant, ctl, seg, ridx0, ridx1, model, metric_log, labels, rank_order (ranking objectives: the rows in
 * the order of the last gradient or metric pass). After tgbm_trainer_boost `gh` may already
 * hold the gradients of the next round (single-tree objectives compute them in the round's last pass). */
size_t tgbm_trainer_get(tgbm_trainer *t, const char *name, void *out, size_t cap);
/* Overwrites gh or y_pred (lock-step tests feed both implementations the same state). */
void tgbm_trainer_set(tgbm_trainer *t, const char *name, const void *in, size_t bytes);

/* Histogram-build timing with HIP events on the trainer's stream. get_profile fills
 * out[0] = summed kernel milliseconds, out[1] = launches, out[2] = rows visited,
 * out[3] = algorithmic bytes (rows x (features + 8 [+4 below the root])). */
void tgbm_trainer_set_profiling(tgbm_trainer *t, int on);
void tgbm_trainer_get_profile(tgbm_trainer *t, double *out4);
/* Per-stage timing of the rounds boosted while profiling was on (the reference accumulates host timers for histogram
 * build, evaluation and data partitioning under its `profiling` switch, hist_tree_builder_single.cu:19-27, :196-219,
 * :392, :400-418; thundergbm_train.cpp:28-30). HIP events on the trainer's stream close every stage. Fills up to
 * `cap` of: out[0] rounds; milliseconds of out[1] gradients + tree init, [2] histogram build, [3] merge + sibling
 * subtraction + root sums, [4] split search + tree update, [5] partition, [6] end of tree (prune, prediction update,
 * fused metric and next gradients), [7] metric as a pass of its own, [8] row re-ordering; then the histogram launches
 * of the root level: [9] milliseconds, [10] launches, [11] algorithmic bytes; and of the levels below it: [12], [13],
 * [14]. Returns the number of values it knows (15). */
int tgbm_trainer_get_phase_profile(tgbm_trainer *t, double *out, int cap);

/* Moves the trees built so far into a model handle usable with the Part 1 functions. */
tgbm_model *tgbm_trainer_export_model(tgbm_trainer *t);

/* Predictor::predict_raw (predictor.cu:32-189) with an explicit base score: class-major raw scores,
 * row_size * trees_per_iter floats. */
void tgbm_predict_raw(int row_size, const float *val, const int *row_ptr, const int *col_ptr, tgbm_model *model,
                      int n_trees, int trees_per_iter, float learning_rate, float base_score, float *out);

/* tgbm_predict_raw for callers that cannot allocate device memory (tight serving loops, harnesses that forbid
 * hipMalloc). It has no counterpart in the reference. Same arguments, same scores bit for bit, but no hipMalloc /
 * hipFree / stream creation: the device copies of the rows, the model and the scores live in a file-scope device
 * array of about 34 MiB that every GPU used by the library holds until the process ends (its address is resolved on
 * the first call on a device). Limits per call: row_size <= 65536, stored values <= 2^20,
 * row_size * trees_per_iter <= 2^19, nodes of the trees used <= 2^19 (e.g. 800 trees of depth 8). Returns 0, or 1
 * with a message on stderr when a limit is exceeded (nothing is computed then); malformed input (a null model, a
 * row_ptr that does not ascend, a negative column index) aborts the process with a message, as in every other entry
 * point. Calls share the device's array, which keeps the last call's contents; they are serialised inside one
 * process, and calls from several processes on one GPU do not interfere (every process has its own copy). The work
 * runs on the default stream with synchronous host copies (the call cannot be recorded into a HIP graph) and returns
 * after the scores were copied to `out`. The trees are walked in their 48-byte node form (the packed LDS form of
 * tgbm_predict_raw needs an allocation), so a call takes about twice the device time of tgbm_predict_raw. */
int tgbm_predict_raw_noalloc(int row_size, const float *val, const int *row_ptr, const int *col_ptr,
                             tgbm_model *model, int n_trees, int trees_per_iter, float learning_rate,
                             float base_score, float *out);

/* Device memory that calls have given back is kept for later ones, at most a 32nd of each GPU's memory; this returns
 * all of it to the driver. It has no counterpart in the reference. */
void tgbm_release_memory(void);

/* Cut points and global bin ids of a CSR matrix (HistCut::get_cut_points_single, hist_cut.cu:232-286;
 * get_bin_ids, hist_tree_builder_single.cu:49-130), computed on the GPU. cut_val / cut_fid need one
 * slot per stored value at most (row_ptr[row_size]); returns the number of cut points. */
int tgbm_cut_points(int row_size, int n_features, const float *val, const int *row_ptr, const int *col_ptr,
                    int max_num_bin, float *cut_val, int *cut_row_ptr, int *cut_fid, int *bin_id);

/* ------------------------------------------------------- Part 3: operators on class scores
 *
 * They work on class scores that lie on the GPU (every pointer in this part is a device pointer of the current device,
 * but for those to the structs themselves), go to the stream that they are given (a hipStream_t; NULL: the default stream), allocate nothing,
 * wait for nothing and can be recorded into a HIP graph. Outputs do not depend on what else runs. They return 0, or 1
 * with a message on stderr when an argument is refused (nothing is launched then), or 2 when a launch failed.
 * They have no counterpart in the reference. */

#define TGBM_F32 0
#define TGBM_F16 1
#define TGBM_BF16 2

/* The score of class c in row i is data[c * class_stride + i * row_stride]; one of the strides is 1: row_stride where the
 * rows of a class lie side by side, as trainers and predictors hold them, class_stride where the classes of a row do. 1 to
 * 2^22 classes. */
typedef struct tgbm_scores {
    const void *data;
    long long class_stride, row_stride;
    int type; /* TGBM_F32, TGBM_F16, TGBM_BF16 */
    int classes, rows;
} tgbm_scores;

/* What is known besides the scores. s = score + bias[class]; a class that the row was shown m > 0 times:
 * s = (s > 0 ? s / repetition : s * repetition) - frequency * m - presence; a class that is not allowed: -infinity,
 * whatever its score is. Each step is one operation in 32 bits.
 * allowed: [allowed_sets][(classes + 31) / 32] words, bit c % 32 of word c / 32 says whether class c is allowed;
 * allowed_set: the rows' sets, a negative number allows everything, one that is no set's nothing; without it there is one
 * set for all rows, or one for each. shown: the rows' lists one behind the other, n_shown classes in all; row i's is
 * [shown_begin[i], shown_begin[i + 1]); numbers that are no classes are skipped. Parts that are NULL are left out. */
typedef struct tgbm_score_rules {
    const float *bias;
    const unsigned *allowed;
    const int *allowed_set;
    const int *shown;
    const long long *shown_begin;
    long long n_shown;
    int allowed_sets;
    float repetition, frequency, presence;
} tgbm_score_rules;

/* out = the scores as the rules leave them, rounded once to their type. out: another array of the same type, classes and
 * rows, in either order, that shares no element with `in`, or `in` itself. */
int tgbm_scores_adjust(const tgbm_scores *in, const tgbm_score_rules *rules, const tgbm_scores *out, void *stream);

/* The k (1 to 128) best classes of every row by the scores as the rules leave them, and the logarithm of the sum of
 * exp(score / temperature) over all classes: exp(value / temperature - lse) is a listed class's probability. values and
 * classes are [rows][k], the best first, of equal scores the lower class; a class whose score is -infinity or NaN is not
 * listed, and what is left of a list is class -1 with -infinity. lse, [rows], is -infinity where nothing is allowed and
 * NaN where a score is that is not taken out. It is a 32-bit number: where value / temperature is large, probabilities from it are off by up to 2^-23 of that
 * (value / temperature of 1000: one part in 8000). temperature: 1e-6 to 1e6. workspace: as many bytes as
 * tgbm_scores_top_workspace says, whose only use is during the call's work on the stream. */
size_t tgbm_scores_top_workspace(const tgbm_scores *in, int k);
int tgbm_scores_top(const tgbm_scores *in, const tgbm_score_rules *rules, int k, float temperature, float *values, int *classes,
                    float *lse, void *workspace, size_t workspace_bytes, void *stream);

/* A teacher's best scores: [rows][entries] (1 to 128) classes and scores, in any order, as tgbm_scores_top lists them.
 * Entries whose class is negative or no class of the student, or whose score is -infinity, are left out; entries that name the
 * same class add up. lse (may be NULL): the logarithm of the sum of exp(score / temperature) over all of the teacher's classes. */
typedef struct tgbm_teacher {
    const int *classes;
    const void *scores;
    const float *lse;
    int type; /* of scores */
    int entries;
} tgbm_teacher;

/* The loss of class scores z against a teacher t, and the gradient pairs for the trees of the next boosting round.
 * With p = softmax(z / T) and the teacher's q = exp(t / T) over their sum, or exp(t / T - lse) where lse is given:
 *   loss = weight * T^2 * [ sum of q (log q - log p) + r (log r - log R) ] + (1 - weight) * -log softmax(z)[label]
 * r = 1 - sum of q (not below 0) is what the teacher left to the classes that it does not name, taken together, R their p;
 * without lse, or where every class is named or the others' scores are all -infinity, there is no such part. A row without entries has no first part,
 * one whose label is no class's number no second.
 *   gradient = weight * T * (M p - q) + (1 - weight) * (softmax(z) - [label]), q of a class that is not named being r p / R
 *   hessian = max(2 (weight * M p (1 - p) + (1 - weight) * s (1 - s)), 1e-16), s = softmax(z): the factor of two and the
 * least value are those of the objective multi:softmax (multiclass_obj.cu:6-35).
 * M = sum of q + r is 1, but with an lse where there is no part for r (M = sum of q), or where the sum of q is above 1.
 * Where all scores of a row are -infinity every p is 0; a NaN or an infinite score or teacher's score makes its row NaN.
 * Everything is 32 bits: terms of the size of log(classes) cancel in the loss of a student that is near its teacher, so about T^2 * 1e-6 of it is rounding;
 * with an lse, q is off by up to 2^-23 of score / T, and so is M where no class takes r. A q below 1e-38 is not counted in the loss.
 * in: float scores, the rows of a class side by side. labels (NULL only where weight is 1): [rows] class numbers as floats. loss (may be NULL): [rows].
 * pairs (may be NULL): gradient and hessian of class c in row i at pairs[2 * (c * pair_stride + i)]. temperature: 1e-3 to
 * 1e3, weight: 0 to 1. workspace: as for tgbm_scores_top. */
size_t tgbm_scores_distill_workspace(const tgbm_scores *in, int entries);
int tgbm_scores_distill(const tgbm_scores *in, const tgbm_teacher *teacher, const float *labels, float temperature, float weight,
                        float *loss, float *pairs, long long pair_stride, void *workspace, size_t workspace_bytes, void *stream);

/* The boosting rounds of a session (Part 2) with a multi:softmax or multi:softprob objective from here on train on that loss:
 * tgbm_trainer_boost and tgbm_trainer_gradient take their gradient pairs from it, with the session's labels. Here the teacher's arrays are
 * host arrays, in the order of the session's rows, classes being numbers of the session's ascending distinct labels; they
 * are copied. NULL: on the labels alone again. Metrics stay those of the labels. Wrong arguments abort the process, as in Part 2. */
void tgbm_trainer_set_teacher(tgbm_trainer *t, const tgbm_teacher *teacher, float temperature, float weight);
/* The mean of that loss over the rows with the current predictions. */
double tgbm_trainer_teacher_loss(tgbm_trainer *t);

/* The scores of a model with one tree per class and round (tgbm_predict_raw with a base score of 0), as the rules leave them, and
 * the best classes by them. Here every pointer, those in the rules among them, is a host pointer, rows are CSR as in
 * sparse_predict_scikit, and calls block until the results are there. adjusted: [trees_per_iter][row_size]; the
 * other outputs as tgbm_scores_top writes them. Wrong arguments abort the process, as in Part 1. */
void tgbm_predict_adjusted(int row_size, const float *val, const int *row_ptr, const int *col_ptr, tgbm_model *model, int n_trees,
                           int trees_per_iter, float learning_rate, const tgbm_score_rules *rules, float *adjusted);
void tgbm_predict_top(int row_size, const float *val, const int *row_ptr, const int *col_ptr, tgbm_model *model, int n_trees,
                      int trees_per_iter, float learning_rate, const tgbm_score_rules *rules, int k, float temperature, float *values,
                      int *classes, float *lse);

#ifdef __cplusplus
}
#endif
#endif /* THUNDERGBM_H */
